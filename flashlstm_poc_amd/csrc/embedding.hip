// Embedding of tokens with a scale, and its gradient by sorted tokens (lm_ops.h).
//
// Both are bound by memory.  The lookup copies rows; a thread takes vectors of eight, whatever the width, so that no lane idles where
// a row is no multiple of a wave.  The gradient sorts the tokens with their positions (stable, eight to ten bits of the token at a
// time), after which the rows of one token lie behind one another: chunks of the sorted list are summed in registers, in the order of the
// positions, and written once where a token's rows end.  What crosses a chunk's border is left as partial sums that a last
// kernel adds up in order.  No atomics on values: the result depends on tokens and sizes alone.
#include "lm_device.h"

namespace flstm_hip {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 32;   // sorted positions a thread sums

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

// ---- the lookup

struct Lookup {
    Tokens t;
    unsigned vectors;   // a row
    size_t first, items, width, ld;
    const void* table;
    void* out;
    float scale;
};

template <class From, class To> __global__ __launch_bounds__(kThreads) void lookup_kernel(Lookup a) {
    const size_t item = a.first + size_t(blockIdx.x) * kThreads + threadIdx.x;
    if (item >= a.items) return;
    const size_t row = item / a.vectors;
    const size_t c = (item - row * a.vectors) * 8;
    const unsigned token = token_at(a.t, row);
    const int n = a.width - c < 8 ? int(a.width - c) : 8;
    float8 v = 0.f;
    if (token < a.t.vocabulary) v = a.scale * load8(static_cast<const From*>(a.table) + token * a.ld + c, n);
    store8(static_cast<To*>(a.out) + row * a.width + c, v, n);
}

// ---- sorting: one stable pass over some bits of the token.  A workgroup has a tile of consecutive entries, each of its waves a
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

__global__ __launch_bounds__(kSortThreads) void count_kernel(SortPass a) {
    __shared__ unsigned counts[1 << kMaxBits];
    const unsigned bins = 1u << a.bits, begin = blockIdx.x * a.tile, end = a.count - begin < a.tile ? a.count : begin + a.tile;
    for (unsigned b = threadIdx.x; b < bins; b += kSortThreads) counts[b] = 0;
    __syncthreads();
    for (unsigned i = begin + threadIdx.x; i < end; i += kSortThreads) atomicAdd(&counts[key_at(a, i) >> a.shift & (bins - 1)], 1u);
    __syncthreads();
    for (unsigned b = threadIdx.x; b < bins; b += kSortThreads) a.counts[size_t(blockIdx.x) * bins + b] = counts[b];
}

__global__ __launch_bounds__(kSortThreads) void scatter_kernel(SortPass a) {
    __shared__ unsigned place[kSortWaves][1 << kMaxBits];   // counts of each wave's part, then where its next entry goes
    __shared__ unsigned sums[kSortThreads];
    const unsigned bins = 1u << a.bits, wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const unsigned begin = blockIdx.x * a.tile, end = a.count - begin < a.tile ? a.count : begin + a.tile;
    const unsigned part = a.tile / kSortWaves, from = begin + wave * part;
    const unsigned to = from >= end ? from : end - from < part ? end : from + part;
    for (unsigned b = lane; b < bins; b += kWave) place[wave][b] = 0;
    for (unsigned i = from + lane; i < to; i += kWave) atomicAdd(&place[wave][key_at(a, i) >> a.shift & (bins - 1)], 1u);
    // entries of a bin in the tiles in front, and in all of them; a thread has `per` consecutive bins
    const unsigned per = (bins + kSortThreads - 1) / kSortThreads;
    unsigned before[(1 << kMaxBits) / kSortThreads], total[(1 << kMaxBits) / kSortThreads], all = 0;
#pragma unroll
    for (unsigned j = 0; j < (1 << kMaxBits) / kSortThreads; ++j) {
        before[j] = total[j] = 0;
        const unsigned b = threadIdx.x * per + j;
        if (j < per && b < bins)
            for (unsigned tile = 0; tile < a.tiles; ++tile) {
                const unsigned n = a.counts[size_t(tile) * bins + b];
                total[j] += n;
                before[j] += tile < blockIdx.x ? n : 0;
            }
        all += total[j];
    }
    sums[threadIdx.x] = all;
    __syncthreads();
    for (unsigned d = 1; d < kSortThreads; d *= 2) {
        const unsigned v = threadIdx.x >= d ? sums[threadIdx.x - d] : 0;
        __syncthreads();
        sums[threadIdx.x] += v;
        __syncthreads();
    }
    unsigned at = sums[threadIdx.x] - all;
#pragma unroll
    for (unsigned j = 0; j < (1 << kMaxBits) / kSortThreads; ++j) {
        const unsigned b = threadIdx.x * per + j;
        if (j < per && b < bins) {
            unsigned next = at + before[j];
#pragma unroll
            for (int w = 0; w < kSortWaves; ++w) {
                const unsigned n = place[w][b];
                place[w][b] = next;
                next += n;
            }
        }
        at += total[j];
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
    unsigned count, vocabulary, vectors, chunks;
    size_t width, ldd;
    const unsigned *keys, *at;
    const void* d_out;
    void* d_table;
    float* partials;   // [chunk][entries of a token that began before; of one that goes on behind][width]
    float scale;
    unsigned sum_blocks;
};

constexpr int kZeroRows = 64;   // rows of the table that a workgroup looks for among the tokens

template <class From, class To> __global__ __launch_bounds__(kThreads) void sum_kernel(Sums a) {
    if (blockIdx.x >= a.sum_blocks) {   // rows without a token
        __shared__ int empty[kZeroRows];
        const size_t row0 = size_t(blockIdx.x - a.sum_blocks) * kZeroRows;
        if (threadIdx.x < kZeroRows) {
            const unsigned row = unsigned(row0) + threadIdx.x;
            unsigned lo = 0, hi = a.count;   // the first entry whose token is not below the row
            while (lo < hi) {
                const unsigned mid = lo + (hi - lo) / 2;
                if (a.keys[mid] < row) lo = mid + 1; else hi = mid;
            }
            empty[threadIdx.x] = row < a.vocabulary && (lo == a.count || a.keys[lo] != row);
        }
        __syncthreads();
        const float8 zero = 0.f;
        for (unsigned i = threadIdx.x; i < kZeroRows * a.vectors; i += kThreads) {
            const unsigned r = i / a.vectors;
            const size_t c = size_t(i - r * a.vectors) * 8;
            if (empty[r]) store8(static_cast<To*>(a.d_table) + (row0 + r) * a.width + c, zero, a.width - c < 8 ? int(a.width - c) : 8);
        }
        return;
    }
    const size_t item = size_t(blockIdx.x) * kThreads + threadIdx.x;
    const unsigned chunk = unsigned(item / a.vectors);
    if (chunk >= a.chunks) return;
    const size_t c = (item - size_t(chunk) * a.vectors) * 8;
    const int n = a.width - c < 8 ? int(a.width - c) : 8;
    const unsigned begin = chunk * kChunk, end = a.count - begin < kChunk ? a.count : begin + kChunk;
    const From* d = static_cast<const From*>(a.d_out) + c;
    To* out = static_cast<To*>(a.d_table) + c;
    float* partial = a.partials + size_t(chunk) * 2 * a.width + c;
    unsigned token = a.keys[begin];
    bool began = begin == 0 || a.keys[begin - 1] != token;   // the token's entries begin in this chunk
    float8 sum = 0.f;
    for (unsigned i = begin; i < end; ++i) {
        const unsigned next = a.keys[i];
        if (next != token) {
            if (began) store8(out + size_t(token) * a.width, a.scale * sum, n);
            else store8(partial, sum, n);
            began = true;
            token = next;
            sum = 0.f;
        }
        if (token >= a.vocabulary) return;
        sum += load8(d + a.at[i] * a.ldd, n);
    }
    const bool ends = end == a.count || a.keys[end] != token;
    if (began && ends) store8(out + size_t(token) * a.width, a.scale * sum, n);
    else store8(partial + (began ? a.width : 0), sum, n);
}

// What each token's entries left in more than one chunk: the chunk that they begin in adds them up.
template <class To> __global__ __launch_bounds__(kThreads) void join_kernel(Sums a) {
    const size_t item = size_t(blockIdx.x) * kThreads + threadIdx.x;
    unsigned chunk = unsigned(item / a.vectors);
    if (chunk + 1 >= a.chunks) return;   // (the last one's end)
    const size_t c = (item - size_t(chunk) * a.vectors) * 8;
    const int n = a.width - c < 8 ? int(a.width - c) : 8;
    const unsigned begin = chunk * kChunk, last = begin + kChunk - 1, token = a.keys[last];
    if (token >= a.vocabulary || a.keys[last + 1] != token || (begin > 0 && a.keys[begin - 1] == token && a.keys[begin] == token)) return;
    const float* partial = a.partials + c;
    float8 sum = load8(partial + (size_t(chunk) * 2 + 1) * a.width, n);
    do {
        ++chunk;
        sum += load8(partial + size_t(chunk) * 2 * a.width, n);
    } while (chunk + 1 < a.chunks && a.keys[chunk * kChunk + kChunk] == token);
    store8(static_cast<To*>(a.d_table) + size_t(token) * a.width + c, a.scale * sum, n);
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
    const size_t tile = round_up(ceil_div(p->tokens, 256), kSortThreads);
    s.tile = unsigned(tile < 2048 ? 2048 : tile);
    s.tiles = unsigned(ceil_div(p->tokens, s.tile));
    return s;
}
struct Room {   // of the workspace, in bytes
    size_t list, counts, partials;
    size_t all() const { return 4 * list + counts + partials; }
};
Room room_of(const flstm_embedding* p) {
    const SortPlan s = sort_plan(p);
    return Room{round_up(p->tokens * 4, 16), round_up((size_t(s.tiles) << s.bits) * 4, 16), round_up(ceil_div(p->tokens, kChunk) * 2 * p->width * 4, 16)};
}

}  // namespace
}  // namespace flstm_hip

using namespace flstm_hip;

extern "C" int flstm_embedding_forward(const flstm_embedding* p, const void* table, size_t ld, flstm_op_dtype table_dtype, void* out,
                                       flstm_op_dtype dtype, void* stream) {
    if (!valid(p) || !valid_dtype(table_dtype) || !valid_dtype(dtype) || (ld < p->width && p->vocabulary > 1)) return FLSTM_E_INVALID;
    if (p->tokens == 0 || p->width == 0) return 0;
    if (!table || !out) return FLSTM_E_INVALID;
    Lookup a{tokens_of(p), unsigned(ceil_div(p->width, 8)), 0, 0, p->width, ld, table, out, p->scale};
    a.items = p->tokens * a.vectors;
    return with_type(table_dtype, [&](auto from) {
        return with_type(dtype, [&](auto to) {
            constexpr size_t kMost = size_t(1) << 31;   // threads a launch
            for (a.first = 0; a.first < a.items; a.first += kMost) {
                const size_t some = a.items - a.first < kMost ? a.items - a.first : kMost;
                lookup_kernel<decltype(from), decltype(to)><<<unsigned(ceil_div(some, kThreads)), kThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
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
    Sums a{};
    a.count = unsigned(p->tokens); a.vocabulary = unsigned(p->vocabulary); a.vectors = unsigned(ceil_div(p->width, 8));
    a.chunks = unsigned(ceil_div(p->tokens, kChunk)); a.width = p->width; a.ldd = ldd; a.d_out = d_out; a.d_table = d_table; a.scale = p->scale;
    const size_t sums = ceil_div(size_t(a.chunks) * a.vectors, kThreads), zeros = ceil_div(p->vocabulary, kZeroRows);
    if (sums + zeros > (size_t(1) << 31) / kThreads * 2 - 1) return FLSTM_E_TOO_LARGE;
    if (p->tokens > 0) {
        const SortPlan plan = sort_plan(p);
        const Room room = room_of(p);
        char* at = static_cast<char*>(workspace);
        unsigned* lists[2][2];
        for (auto& pair : lists)
            for (auto& list : pair) {
                list = reinterpret_cast<unsigned*>(at);
                at += room.list;
            }
        SortPass pass{tokens_of(p), a.count, plan.tile, plan.tiles, 0, plan.bits, 1, nullptr, nullptr, nullptr, nullptr, reinterpret_cast<unsigned*>(at)};
        a.partials = reinterpret_cast<float*>(at + room.counts);
        for (int i = 0; i < plan.passes; ++i) {
            pass.shift = i * plan.bits;
            pass.first = i == 0;
            pass.keys_in = lists[(i + 1) % 2][0]; pass.at_in = lists[(i + 1) % 2][1];
            pass.keys_out = lists[i % 2][0]; pass.at_out = lists[i % 2][1];
            count_kernel<<<plan.tiles, kSortThreads, 0, s>>>(pass);
            scatter_kernel<<<plan.tiles, kSortThreads, 0, s>>>(pass);
            if (const int rc = launched()) return rc;
        }
        a.keys = lists[(plan.passes + 1) % 2][0]; a.at = lists[(plan.passes + 1) % 2][1];
    }
    a.sum_blocks = unsigned(sums);
    return with_type(dtype, [&](auto from) {
        return with_type(table_dtype, [&](auto to) {
            sum_kernel<decltype(from), decltype(to)><<<unsigned(sums + zeros), kThreads, 0, s>>>(a);
            if (const int rc = launched()) return rc;
            if (a.chunks > 1) join_kernel<decltype(to)><<<unsigned(sums), kThreads, 0, s>>>(a);
            return launched();
        });
    });
}
