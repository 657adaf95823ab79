// Embedding of tokens with a scale, and its gradient by sorted tokens (lm_ops.h).
//
// Both are bound by memory.  The lookup copies rows; a thread takes vectors of sixteen bytes, whatever the width, so that no lane idles where
// a row is no multiple of a wave.  The gradient sorts the tokens with their positions, stable, after which the rows of one token lie behind one
// another: chunks of the sorted list are summed in registers, in the order of the positions, and written once where a token's rows end.  What
// crosses a chunk's border is put together in LDS by the workgroup, whose chunks follow each other, and what crosses the workgroup's is left as partial
// sums that a last kernel adds up in order.  No atomics on values: the result depends on tokens and sizes alone.
// Few tokens are sorted by counting for each how many come in front of it, in one launch; many in stable passes over at most ten bits.
// 65536 tokens of a text, 1024 fp16 channels, 50001 fp32 rows: lookup 38 us, 7.1 TB/s with what the caches hold of the table; sort 40, which writes
// 205 MB of zeros meanwhile, 5.1 TB/s; sums 44, 4.6 TB/s; partial sums 5.
#include <algorithm>
#include <type_traits>

#include "lm_device.h"

namespace flstm_hip {
namespace {

constexpr int kThreads = 256;

struct Tokens {
    size_t count;
    unsigned vocabulary;
    const void* index;
    int index_64;
};
// Token i, `vocabulary` for all that lie outside.
__device__ __forceinline__ unsigned token_at(const Tokens& t, size_t i) {
    const long long v = t.index_64 ? static_cast<const long long*>(t.index)[i] : static_cast<const int*>(t.index)[i];
    return v >= 0 && v < (long long)t.vocabulary ? unsigned(v) : t.vocabulary;
}

// Rows are taken in vectors of N columns, sixteen bytes of what is read or written most, so that a wave's request is one piece; vector v is N columns from
// the returned one on, which the last two of a width that is no multiple of N have in part in common: what is common is computed and written twice, alike.
// So no lane has a branch of its own, behind which its loads would be waited for one by one.  Rows of less than a vector are taken column by column.
template <class T> constexpr int kVector = 16 / int(sizeof(T));
template <int N> using Floats = float __attribute__((ext_vector_type(N)));
template <int N> __device__ __forceinline__ size_t column(size_t v, size_t width) { return v * N + N <= width ? v * N : width - N; }
template <bool kPassing, class V, class T> __device__ __forceinline__ void store_any(T* p, V v) {
    typedef V __attribute__((aligned(sizeof(T)))) U;
    if constexpr (kPassing) __builtin_nontemporal_store(v, reinterpret_cast<U*>(p));
    else *reinterpret_cast<U*>(p) = v;
}
template <int N, bool kPassing, class T> __device__ __forceinline__ Floats<N> load_vector(const T* p) {
    typedef T V __attribute__((ext_vector_type(N)));
    typedef V __attribute__((aligned(sizeof(T)))) U;
    if constexpr (kPassing) return __builtin_convertvector(__builtin_nontemporal_load(reinterpret_cast<const U*>(p)), Floats<N>);
    else return __builtin_convertvector(*reinterpret_cast<const U*>(p), Floats<N>);
}
template <int N, bool kPassing, class T> __device__ __forceinline__ void store_vector(T* p, Floats<N> v) {
    typedef T V __attribute__((ext_vector_type(N)));
    store_any<kPassing>(p, __builtin_convertvector(v, V));
}
// Beyond what the L2s hold, looked-up rows and the gradient's zeros are written past them (kPassing): 65536 rows of 1024 fp16 are looked up in 39 us instead of
// 48.  What the gradient sums is read past them from half of what the cache behind them holds on, where rows begin with lines: 131072 rows of 1024 fp16
// are summed in 76 us instead of 80, 200000 in 105 instead of 110, and what comes behind is as much faster again; but rows of 1000, whose lines two workgroups share, take 99
// instead of 86, and 60000 of 512 fp32, which that cache holds, 27 instead of 24.
constexpr size_t kMostKept = size_t(32) << 20, kMostRead = size_t(128) << 20, kLine = 128;   // bytes

// ---- the lookup

constexpr int kLookups = 2;   // vectors a thread has on their way

struct Lookup {
    Tokens t;
    unsigned vectors, items;   // a row; a launch
    size_t first, width, ld;   // first: the launch's first row
    const void* table;
    void* out;
    float scale;
};

// (fp32 results in vectors of eight, whose two stores each leave every other sixteen bytes, past the L2: 60000 rows of 500 in 44 us instead of 20.)
template <class From, class To, int N, bool kPassing> __global__ __launch_bounds__(kThreads) void lookup_kernel(Lookup a) {
    unsigned token[kLookups];
    To* out[kLookups];
    Floats<N> v[kLookups];
    const unsigned item = blockIdx.x * (kThreads * kLookups) + threadIdx.x;
    const auto there = [&](int j) { return item + j * kThreads < a.items; };
#pragma unroll
    for (int j = 0; j < kLookups; ++j) {
        const unsigned i = there(j) ? item + j * kThreads : 0, r = i / a.vectors;
        const size_t row = a.first + r, c = column<N>(i - r * a.vectors, a.width);
        token[j] = token_at(a.t, row);
        out[j] = static_cast<To*>(a.out) + row * a.width + c;
        v[j] = load_vector<N, false>(static_cast<const From*>(a.table) + (token[j] < a.t.vocabulary ? token[j] : 0) * a.ld + c);
    }
#pragma unroll
    for (int j = 0; j < kLookups; ++j) {
        const Floats<N> zero = 0.f;
        if (there(j)) store_vector<N, kPassing>(out[j], token[j] < a.t.vocabulary ? a.scale * v[j] : zero);
    }
}

// ---- zeros for the whole gradient, of which the tokens' rows are written afterwards.  Sorting leaves most of the chip idle: each of its launches has
// workgroups behind its own that clear a share of the table meanwhile.  (Clearing only what has no token, beside the sums, is a third fewer bytes and a search
// for every row, and takes 89 us instead of 87 for sorting 65536 tokens and the sums of 1024 fp16 over 50001 fp32 rows.)

struct Zeros {
    char* at;
    size_t bytes;          // of the launch's share
    unsigned first;        // the launch's first workgroup for this
};
constexpr size_t kZeroBytes = 65536;   // a workgroup

template <bool kPassing> __device__ __forceinline__ void clear_share(const Zeros& z) {
    const size_t begin = size_t(blockIdx.x - z.first) * kZeroBytes, end = z.bytes - begin < kZeroBytes ? z.bytes : begin + kZeroBytes;
    typedef unsigned Piece __attribute__((ext_vector_type(4)));
    const Piece zero = 0u;
    if (z.bytes < sizeof(Piece)) {
        if (threadIdx.x < z.bytes / 2) reinterpret_cast<short*>(z.at)[threadIdx.x] = 0;
        return;
    }
    for (size_t i = begin + threadIdx.x * sizeof(Piece); i < end; i += blockDim.x * sizeof(Piece))
        store_any<kPassing>(reinterpret_cast<short*>(z.at + (i + sizeof(Piece) <= z.bytes ? i : z.bytes - sizeof(Piece))), zero);
}

// ---- sorting few tokens: an entry's place is the number of those in front of it.  A workgroup has 64 entries, each of its waves a
// part of all others.

constexpr int kRankThreads = 1024, kRankWaves = kRankThreads / kWave;
constexpr size_t kMostRanked = 8192;

template <bool kPassing> __global__ __launch_bounds__(kRankThreads) void rank_kernel(Tokens t, unsigned* keys_out, unsigned* at_out, Zeros zeros) {
    if (blockIdx.x >= zeros.first) return clear_share<kPassing>(zeros);
    extern __shared__ unsigned keys[];   // all of them, rounded up to whole fours a wave, and kRankWaves rows of kWave counts
    const unsigned count = unsigned(t.count), part = (count + kRankWaves * 4 - 1) / (kRankWaves * 4) * 4, whole = part * kRankWaves;
    unsigned* counts = keys + whole;
    for (unsigned i = threadIdx.x; i < whole; i += kRankThreads) keys[i] = i < count ? token_at(t, i) : ~0u;   // (behind all others)
    __syncthreads();
    const unsigned wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave, first = blockIdx.x * kWave, i = first + lane;
    const unsigned key = i < whole ? keys[i] : ~0u, from = wave * part, to = from + part;
    unsigned rank = 0;
    typedef unsigned uint4v __attribute__((ext_vector_type(4)));
    const auto among = [&](unsigned begin, unsigned end, auto&& ahead) {
        if (begin < from) begin = from;
        if (end > to) end = to;
#pragma unroll 4
        for (unsigned j = begin; j < end; j += 4) {
            const uint4v k = *reinterpret_cast<const uint4v*>(keys + j);
#pragma unroll
            for (int e = 0; e < 4; ++e) rank += ahead(k[e], j + e);
        }
    };
    among(0, first, [&](unsigned k, unsigned) { return k <= key; });
    among(first, first + kWave, [&](unsigned k, unsigned j) { return k < key || (k == key && j < i); });
    among(first + kWave, whole, [&](unsigned k, unsigned) { return k < key; });
    counts[wave * kWave + lane] = rank;
    __syncthreads();
    if (wave == 0 && i < count) {
        rank = 0;
#pragma unroll
        for (int w = 0; w < kRankWaves; ++w) rank += counts[w * kWave + lane];
        keys_out[rank] = key;
        at_out[rank] = i;
    }
}

// ---- sorting many tokens: one stable pass over some bits of the token.  A workgroup has a tile of consecutive entries, each of its waves a
// consecutive part of that, 64 entries at a time in order.

constexpr int kSortThreads = 512, kSortWaves = kSortThreads / kWave, kMaxBits = 10;

struct SortPass {
    Tokens t;
    unsigned count, tile, tiles;
    int shift, bits, first;            // first: keys are the tokens themselves, positions their places
    const unsigned *keys_in, *at_in;
    unsigned *keys_out, *at_out, *counts;   // counts: [tile][1 << bits]
};
__device__ __forceinline__ unsigned key_at(const SortPass& a, unsigned i) { return a.first ? token_at(a.t, i) : a.keys_in[i]; }

template <bool kPassing> __global__ __launch_bounds__(kSortThreads) void count_kernel(SortPass a, Zeros zeros) {
    if (blockIdx.x >= zeros.first) return clear_share<kPassing>(zeros);
    __shared__ unsigned counts[1 << kMaxBits];
    const unsigned bins = 1u << a.bits, begin = blockIdx.x * a.tile, end = a.count - begin < a.tile ? a.count : begin + a.tile;
    for (unsigned b = threadIdx.x; b < bins; b += kSortThreads) counts[b] = 0;
    __syncthreads();
    for (unsigned i = begin + threadIdx.x; i < end; i += kSortThreads) atomicAdd(&counts[key_at(a, i) >> a.shift & (bins - 1)], 1u);
    __syncthreads();
    for (unsigned b = threadIdx.x; b < bins; b += kSortThreads) a.counts[size_t(blockIdx.x) * bins + b] = counts[b];
}

// Adds the tiles' counts of every bin up: those in front of this workgroup's, and all.  A thread has P bins, kSortThreads apart, or where there are fewer bins
// than threads some of the tiles.
template <unsigned P> __device__ __forceinline__ void add_counts(const SortPass& a, unsigned* in_front, unsigned* in_all) {
    constexpr unsigned kAhead = 16;   // tiles on their way together
    const unsigned bins = 1u << a.bits, sharers = bins < kSortThreads ? kSortThreads / bins : 1, b = threadIdx.x % bins;
    unsigned before[P], total[P];
#pragma unroll
    for (unsigned j = 0; j < P; ++j) before[j] = total[j] = 0;
    for (unsigned first = threadIdx.x / bins; first < a.tiles; first += kAhead * sharers) {
        unsigned n[P][kAhead];
#pragma unroll
        for (unsigned k = 0; k < kAhead; ++k)
#pragma unroll
            for (unsigned j = 0; j < P; ++j) {
                const unsigned tile = first + k * sharers;
                n[j][k] = a.counts[size_t(tile < a.tiles ? tile : first) * bins + b + j * kSortThreads];
            }
#pragma unroll
        for (unsigned k = 0; k < kAhead; ++k)
#pragma unroll
            for (unsigned j = 0; j < P; ++j) {
                const unsigned tile = first + k * sharers, v = tile < a.tiles ? n[j][k] : 0;
                total[j] += v;
                before[j] += tile < blockIdx.x ? v : 0;
            }
    }
#pragma unroll
    for (unsigned j = 0; j < P; ++j) {
        if (total[j]) atomicAdd(&in_all[b + j * kSortThreads], total[j]);
        if (before[j]) atomicAdd(&in_front[b + j * kSortThreads], before[j]);
    }
}

template <bool kPassing> __global__ __launch_bounds__(kSortThreads) void scatter_kernel(SortPass a, Zeros zeros) {
    if (blockIdx.x >= zeros.first) return clear_share<kPassing>(zeros);
    __shared__ unsigned place[kSortWaves][1 << kMaxBits];   // counts of each wave's part, then where its next entry goes
    __shared__ unsigned sums[(1 << kMaxBits) / kSortThreads][kSortWaves], in_front[1 << kMaxBits], in_all[1 << kMaxBits];
    const unsigned bins = 1u << a.bits, wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const unsigned begin = blockIdx.x * a.tile, end = a.count - begin < a.tile ? a.count : begin + a.tile;
    const unsigned part = a.tile / kSortWaves, from = begin + wave * part;
    const unsigned to = from >= end ? from : end - from < part ? end : from + part;
    for (unsigned b = lane; b < bins; b += kWave) place[wave][b] = 0;
    for (unsigned i = from + lane; i < to; i += kWave) atomicAdd(&place[wave][key_at(a, i) >> a.shift & (bins - 1)], 1u);
    // entries of a bin in the tiles in front, and in all of them
    constexpr unsigned kPer = (1 << kMaxBits) / kSortThreads;
    for (unsigned b = threadIdx.x; b < bins; b += kSortThreads) in_front[b] = in_all[b] = 0;
    __syncthreads();
    if (bins > kSortThreads) add_counts<kPer>(a, in_front, in_all);
    else add_counts<1>(a, in_front, in_all);
    __syncthreads();
    unsigned before[kPer], total[kPer];
#pragma unroll
    for (unsigned j = 0; j < kPer; ++j) {
        const unsigned b = threadIdx.x + j * kSortThreads;
        before[j] = b < bins ? in_front[b] : 0;
        total[j] = b < bins ? in_all[b] : 0;
    }
    unsigned start = 0;   // of the thread's bins, the entries in all bins in front of the first
#pragma unroll
    for (unsigned j = 0; j < kPer; ++j) {
        const unsigned b = threadIdx.x + j * kSortThreads;
        unsigned at = total[j];   // the sum over the threads up to this one
#pragma unroll
        for (int d = 1; d < kWave; d *= 2) {
            const unsigned v = __shfl_up(at, d);
            at += int(lane) >= d ? v : 0;
        }
        if (lane == kWave - 1) sums[j][wave] = at;
        __syncthreads();
        at += start - total[j];
        unsigned all = 0;
#pragma unroll
        for (unsigned w = 0; w < kSortWaves; ++w) {
            at += w < wave ? sums[j][w] : 0;
            all += sums[j][w];
        }
        start += all;
        if (b < bins) {
            unsigned next = at + before[j];
#pragma unroll
            for (int w = 0; w < kSortWaves; ++w) {
                const unsigned n = place[w][b];
                place[w][b] = next;
                next += n;
            }
        }
    }
    __syncthreads();
    // (the loop's count is the wave's own, so that all its lanes take part in the ballots)
    for (unsigned base = from; base < to; base += kWave) {
        const unsigned i = base + lane;
        const bool there = i < to;
        const unsigned key = there ? key_at(a, i) : 0, position = there ? (a.first ? i : a.at_in[i]) : 0;
        const unsigned digit = key >> a.shift & (bins - 1);
        u64 same = __ballot(there);
        for (int b = 0; b < a.bits; ++b) {
            const u64 set = __ballot(digit >> b & 1);
            same &= (digit >> b & 1) ? set : ~set;
        }
        const unsigned rank = __popcll(same & ((u64(1) << lane) - 1)), many = __popcll(same);
        unsigned first = 0;
        if (there) first = place[wave][digit];
        __builtin_amdgcn_wave_barrier();
        if (there && rank == 0) place[wave][digit] = first + many;
        __builtin_amdgcn_wave_barrier();
        if (there) {
            a.keys_out[first + rank] = key;
            a.at_out[first + rank] = position;
        }
    }
}

// ---- the gradient from sorted tokens

struct Sums {
    unsigned count, vocabulary, vectors, groups, slabs;   // groups: of kThreads / LANES chunks; slabs: of LANES vectors
    int chunk;                                            // entries
    size_t width, ldd;
    const unsigned *keys, *at;
    const void* d_out;
    void* d_table;
    float* partials;   // [group][entries of a token that began before; of one that goes on behind][width]
    float scale;
};

constexpr int kMaxChunk = 32;

// A thread sums the entries of one chunk in one vector of columns; kThreads / LANES chunks behind one another and LANES vectors beside one
// another are a workgroup's.
template <class From, class To, int N, int LANES, bool kPassing> __global__ __launch_bounds__(kThreads) void sum_kernel(Sums a) {
    constexpr int kChunks = kThreads / LANES, kRows = 8;   // rows on their way to a thread
    __shared__ unsigned keys[kChunks * kMaxChunk + 2], at[kChunks * kMaxChunk];   // keys: with those in front of and behind the workgroup's
    __shared__ Floats<N> heads[kChunks][LANES], tails[kChunks][LANES];
    const unsigned group = blockIdx.x / a.slabs, slab = blockIdx.x - group * a.slabs;
    const int size = kChunks * a.chunk, tid = threadIdx.x, chunk = tid / LANES;
    int lane = tid % LANES;
    const unsigned begin = group * size;
    const int here = a.count - begin < unsigned(size) ? int(a.count - begin) : size;
    constexpr unsigned kNone = ~0u;   // no token, and not the one behind the vocabulary
#pragma unroll
    for (int j = 0; j < kChunks * kMaxChunk / kThreads; ++j) {
        const int i = tid + j * kThreads;
        const unsigned from = i < here ? begin + i : begin;   // (any entry, where there is none)
        const unsigned key = a.keys[from], place = a.at[from];
        if (i < size) {
            keys[i + 1] = i < here ? key : kNone;
            at[i] = place;
        }
    }
    if (tid < 2) {
        const bool there = tid == 0 ? group > 0 : begin + size < a.count;
        keys[tid == 0 ? 0 : size + 1] = there ? a.keys[tid == 0 ? begin - 1 : begin + size] : kNone;
    }
    __syncthreads();
    if (slab * LANES + lane >= a.vectors) lane = a.vectors - 1 - slab * LANES;   // (a slab's last lanes do the last one's work again)
    const size_t c = column<N>(slab * LANES + lane, a.width);
    const From* d = static_cast<const From*>(a.d_out) + c;
    To* out = static_cast<To*>(a.d_table) + c;
    const auto put = [&](unsigned row, Floats<N> v) { store_vector<N, false>(out + size_t(row) * a.width, a.scale * v); };
    const unsigned* key = keys + 1;
    const int from = chunk * a.chunk, to = from + a.chunk;
    unsigned token = key[from];
    Floats<N> sum = 0.f;
    bool began = key[from - 1] != token;   // the token's entries begin in this chunk
    for (int i = from; i < to; i += kRows) {
        Floats<N> row[kRows];
        unsigned next[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            next[r] = key[i + r];
            row[r] = load_vector<N, kPassing>(d + at[i + r] * a.ldd);
        }
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            if (next[r] != token) {
                if (!began) heads[chunk][lane] = sum;
                else if (token < a.vocabulary) put(token, sum);
                began = true;
                token = next[r];
                sum = 0.f;
            }
            sum += row[r];
        }
    }
    if (began && key[to] != token) {
        if (token < a.vocabulary) put(token, sum);
    } else if (began) {
        tails[chunk][lane] = sum;
    } else {
        heads[chunk][lane] = sum;
    }
    __syncthreads();
    // what crosses the chunks' borders, in order
    if (chunk > 0) return;
    sum = 0.f;
    began = false;
    float* partial = a.partials + size_t(group) * 2 * a.width + c;
#pragma unroll 4
    for (int k = 0; k < kChunks; ++k) {
        const int first = k * a.chunk, last = first + a.chunk - 1;
        const unsigned front = key[first - 1], head = key[first], tail = key[last], behind = key[last + 1];
        const Floats<N> of_head = heads[k][lane], of_tail = tails[k][lane];
        const bool enters = head < a.vocabulary && front == head, leaves = tail < a.vocabulary && behind == tail, whole = enters && head == tail;
        if (enters) sum += of_head;
        if (enters && !(whole && leaves)) {
            if (began) put(head, sum);
            else store_vector<N, false>(partial, sum);
        }
        if (leaves && !whole) {
            sum = of_tail;
            began = true;
        }
    }
    const unsigned tail = key[size - 1];
    if (tail < a.vocabulary && key[size] == tail) store_vector<N, false>(partial + (began ? a.width : 0), sum);
}

// What each token's entries left in more than one group: the group that they begin in adds them up.
template <class To, int N> __global__ __launch_bounds__(kThreads) void join_kernel(Sums a, unsigned size) {
    const unsigned item = blockIdx.x * kThreads + threadIdx.x;
    unsigned group = item / a.vectors;
    if (group + 1 >= a.groups) return;
    const size_t c = column<N>(item - group * a.vectors, a.width);
    const unsigned begin = group * size, last = begin + size - 1, token = a.keys[last];
    if (token >= a.vocabulary || a.keys[last + 1] != token || (begin > 0 && a.keys[begin - 1] == token)) return;
    const float* partial = a.partials + c;
    Floats<N> sum = load_vector<N, false>(partial + (size_t(group) * 2 + 1) * a.width);
    constexpr int kAhead = 8;
    for (bool more = true; more;) {
        Floats<N> v[kAhead];
        bool there[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const unsigned g = group + 1 + j < a.groups ? group + 1 + j : a.groups - 1;
            there[j] = (group + 1 + j < a.groups) & (a.keys[g * size] == token);   // (no branch: all on their way together)
            v[j] = load_vector<N, false>(partial + size_t(g) * 2 * a.width);
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (there[j]) sum += v[j];
        more = there[kAhead - 1];
        group += kAhead;
    }
    store_vector<N, false>(static_cast<To*>(a.d_table) + size_t(token) * a.width + c, a.scale * sum);
}

// ---- host side

bool valid(const flstm_embedding* p) {
    return p && p->vocabulary >= 1 && p->vocabulary < (size_t(1) << 31) && p->tokens < (size_t(1) << 31) && p->width < (size_t(1) << 24) &&
           p->scale == p->scale && (p->tokens == 0 || p->index);
}
Tokens tokens_of(const flstm_embedding* p) { return Tokens{p->tokens, unsigned(p->vocabulary), p->index, p->index_64}; }

// How the tokens are sorted: passes of at most kMaxBits bits, which hold every token and the one behind them; tiles that are as many
// as a workgroup adds up the counts of in passing.
struct SortPlan {
    int passes, bits;
    unsigned tile, tiles;
};
SortPlan sort_plan(const flstm_embedding* p) {
    int bits = 1;
    while (bits < 32 && (p->vocabulary >> bits) != 0) ++bits;
    SortPlan s;
    s.passes = (bits + kMaxBits - 1) / kMaxBits;
    s.bits = (bits + s.passes - 1) / s.passes;
    const size_t tile = round_up(ceil_div(p->tokens, 128), kSortThreads);
    s.tile = unsigned(tile < 1024 ? 1024 : tile);
    s.tiles = unsigned(ceil_div(p->tokens, s.tile));
    return s;
}
bool ranked(const flstm_embedding* p) { return p->tokens <= kMostRanked; }

// Lanes beside one another for a row's vectors, and entries a thread sums: as many as leave enough workgroups.
struct SumPlan {
    int vector, lanes, chunk;   // columns; lanes; entries
    unsigned groups, slabs;
    size_t size() const { return size_t(kThreads / lanes) * chunk; }
};
SumPlan sum_plan(const flstm_embedding* p, size_t element) {
    SumPlan s;
    s.vector = p->width * element < 16 ? 1 : int(16 / element);
    const size_t vectors = ceil_div(p->width, size_t(s.vector));
    s.lanes = vectors <= 4 ? 4 : vectors <= 8 ? 8 : 16;
    s.slabs = unsigned(ceil_div(vectors, s.lanes));
    for (s.chunk = kMaxChunk; s.chunk > 8 && ceil_div(p->tokens, s.size()) * s.slabs < 512;) s.chunk /= 2;
    s.groups = unsigned(ceil_div(p->tokens, s.size()));
    return s;
}
struct Room {   // of the workspace, in bytes
    size_t list, lists, counts, partials;
    size_t all() const { return lists * list + counts + partials; }
};
Room room_of(const flstm_embedding* p) {
    const SortPlan s = sort_plan(p);
    return Room{round_up(p->tokens * 4, 16), size_t(ranked(p) ? 2 : 4), ranked(p) ? 0 : round_up((size_t(s.tiles) << s.bits) * 4, 16),
                round_up(std::max(size_t(sum_plan(p, 2).groups), size_t(sum_plan(p, 4).groups)) * 2 * p->width * 4, 16)};   // (of any type)
}

}  // namespace
}  // namespace flstm_hip

using namespace flstm_hip;

extern "C" int flstm_embedding_forward(const flstm_embedding* p, const void* table, size_t ld, flstm_op_dtype table_dtype, void* out,
                                       flstm_op_dtype dtype, void* stream) {
    if (!valid(p) || !valid_dtype(table_dtype) || !valid_dtype(dtype) || (ld < p->width && p->vocabulary > 1)) return FLSTM_E_INVALID;
    if (p->tokens == 0 || p->width == 0) return 0;
    if (!table || !out) return FLSTM_E_INVALID;
    Lookup a{tokens_of(p), 0, 0, 0, p->width, ld, table, out, p->scale};
    return with_type(table_dtype, [&](auto from) {
        return with_type(dtype, [&](auto to) {
            constexpr int N = kVector<decltype(to)>;
            const size_t n = p->width < N ? 1 : N;
            a.vectors = unsigned(ceil_div(p->width, n));
            const size_t most = (size_t(1) << 31) / a.vectors;   // rows a launch
            const bool passing = p->tokens * p->width * sizeof(to) > kMostKept;
            for (a.first = 0; a.first < p->tokens; a.first += most) {
                a.items = unsigned((p->tokens - a.first < most ? p->tokens - a.first : most) * a.vectors);
                const unsigned grid = unsigned(ceil_div(a.items, kThreads * kLookups));
                hipStream_t s = static_cast<hipStream_t>(stream);
                if (n == 1) lookup_kernel<decltype(from), decltype(to), 1, false><<<grid, kThreads, 0, s>>>(a);
                else if (passing) lookup_kernel<decltype(from), decltype(to), N, true><<<grid, kThreads, 0, s>>>(a);
                else lookup_kernel<decltype(from), decltype(to), N, false><<<grid, kThreads, 0, s>>>(a);
                if (const int rc = launched()) return rc;
            }
            return 0;
        });
    });
}

extern "C" size_t flstm_embedding_workspace_bytes(const flstm_embedding* p) { return valid(p) && p->width ? room_of(p).all() : 0; }

extern "C" int flstm_embedding_backward(const flstm_embedding* p, const void* d_out, size_t ldd, flstm_op_dtype dtype, void* d_table,
                                        flstm_op_dtype table_dtype, void* workspace, void* stream) {
    if (!valid(p) || !valid_dtype(table_dtype) || !valid_dtype(dtype)) return FLSTM_E_INVALID;
    if (p->width == 0) return 0;
    if (!d_table || (p->tokens > 0 && (!d_out || !workspace))) return FLSTM_E_INVALID;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const SumPlan plan = sum_plan(p, dtype == FLSTM_OP_F32 ? 4 : 2);
    Sums a{};
    a.count = unsigned(p->tokens); a.vocabulary = unsigned(p->vocabulary); a.vectors = unsigned(ceil_div(p->width, size_t(plan.vector)));
    a.groups = plan.groups; a.slabs = plan.slabs; a.chunk = plan.chunk;
    a.width = p->width; a.ldd = ldd; a.d_out = d_out; a.d_table = d_table; a.scale = p->scale;
    const size_t sums = size_t(a.groups) * a.slabs, joins = ceil_div(size_t(a.groups) * a.vectors, kThreads);
    const size_t size = table_dtype == FLSTM_OP_F32 ? 4 : 2, bytes = p->vocabulary * p->width * size;
    const bool passing = bytes > kMostKept;
    const SortPlan sort = sort_plan(p);
    const int launches = ranked(p) ? 1 : 2 * sort.passes;
    const size_t share = round_up(ceil_div(bytes, launches), kZeroBytes);   // that each clears
    if (sums > 0xffffffffu / kThreads || joins > 0xffffffffu / kThreads || share / kZeroBytes + kMostRanked > 0xffffffffu / kRankThreads) return FLSTM_E_TOO_LARGE;
    int launch = 0;
    const auto zeros_behind = [&](unsigned blocks, unsigned& grid) {
        const size_t from = share * launch++, some = from >= bytes ? 0 : bytes - from < share ? bytes - from : share;
        grid = blocks + unsigned(ceil_div(some, kZeroBytes));
        return Zeros{static_cast<char*>(d_table) + from, some, blocks};
    };
    const Room room = room_of(p);
    char* at = static_cast<char*>(workspace);
    unsigned* lists[2][2] = {};
    for (size_t i = 0; i < room.lists; ++i, at += room.list) lists[i / 2][i % 2] = reinterpret_cast<unsigned*>(at);
    int last = 0;
    unsigned grid;
    if (ranked(p)) {
        const size_t lds = (round_up(p->tokens, kRankWaves * 4) + kRankThreads) * 4;
        const Zeros zeros = zeros_behind(unsigned(ceil_div(p->tokens, kWave)), grid);
        if (passing) rank_kernel<true><<<grid, kRankThreads, lds, s>>>(tokens_of(p), lists[0][0], lists[0][1], zeros);
        else rank_kernel<false><<<grid, kRankThreads, lds, s>>>(tokens_of(p), lists[0][0], lists[0][1], zeros);
    } else {
        SortPass pass{tokens_of(p), a.count, sort.tile, sort.tiles, 0, sort.bits, 1, nullptr, nullptr, nullptr, nullptr, reinterpret_cast<unsigned*>(at)};
        for (int i = 0; i < sort.passes; ++i) {
            last = i % 2;
            pass.shift = i * sort.bits;
            pass.first = i == 0;
            pass.keys_in = lists[1 - last][0]; pass.at_in = lists[1 - last][1];
            pass.keys_out = lists[last][0]; pass.at_out = lists[last][1];
            Zeros zeros = zeros_behind(sort.tiles, grid);
            if (passing) count_kernel<true><<<grid, kSortThreads, 0, s>>>(pass, zeros);
            else count_kernel<false><<<grid, kSortThreads, 0, s>>>(pass, zeros);
            zeros = zeros_behind(sort.tiles, grid);
            if (passing) scatter_kernel<true><<<grid, kSortThreads, 0, s>>>(pass, zeros);
            else scatter_kernel<false><<<grid, kSortThreads, 0, s>>>(pass, zeros);
        }
    }
    if (const int rc = launched()) return rc;
    if (p->tokens == 0) return 0;
    a.keys = lists[last][0]; a.at = lists[last][1];
    a.partials = reinterpret_cast<float*>(at + room.counts);
    return with_type(dtype, [&](auto from) {
        return with_type(table_dtype, [&](auto to) {
            typedef decltype(from) From;
            typedef decltype(to) To;
            const unsigned grid = unsigned(sums);
            const bool passing = p->tokens * p->width * sizeof(From) >= kMostRead && ldd * sizeof(From) % kLine == 0 && reinterpret_cast<uintptr_t>(d_out) % kLine == 0;
            const auto sum = [&](auto lanes, auto vector) {
                constexpr int kLanes = decltype(lanes)::value, N = decltype(vector)::value;
                constexpr bool kPassing = N > 1;   // (not for rows of less than a vector, column by column)
                if (kPassing && passing) sum_kernel<From, To, N, kLanes, kPassing><<<grid, kThreads, 0, s>>>(a);
                else sum_kernel<From, To, N, kLanes, false><<<grid, kThreads, 0, s>>>(a);
                if (const int rc = launched()) return rc;
                if (a.groups > 1) join_kernel<To, N><<<unsigned(joins), kThreads, 0, s>>>(a, unsigned(plan.size()));
                return launched();
            };
            constexpr std::integral_constant<int, kVector<From>> whole;
            constexpr std::integral_constant<int, 1> single;
            if (plan.vector == 1) return plan.lanes == 4 ? sum(std::integral_constant<int, 4>(), single) : sum(std::integral_constant<int, 8>(), single);
            if (plan.lanes == 16) return sum(std::integral_constant<int, 16>(), whole);
            if (plan.lanes == 8) return sum(std::integral_constant<int, 8>(), whole);
            return sum(std::integral_constant<int, 4>(), whole);
        });
    });
}
