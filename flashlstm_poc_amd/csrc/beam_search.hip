// Beam search (lm_ops.h): the best continuations of every sequence's beams, and the beams' states moved behind them.
//
// The selection is bound by one reading of the logits.  A workgroup has a part of a row: the part's largest logit, the sum of its
// exponentials, and its best entries, all from registers.  What takes part in the ordering are whole numbers, the logit's order
// above and the place's complement below, so that no two are equal and equal logits come lowest place first; the k-th best of the
// threads' own best entries is a bound that at least k entries reach, and only the k threads in front of it can hold others that
// do.  A second kernel puts the parts together: the rows' logarithms, and the candidates' values in 64 bits, so that which of two
// is larger does not depend on a rounding to 32.
#include "lm_device.h"

namespace flstm_hip {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxKeep = 32, kMaxBeams = 32;
constexpr int kVectors = 4, kTile = kThreads * kVectors * 8;   // logits a workgroup holds at a time
constexpr size_t kMaxParts = 64;
constexpr float kLowest = -3.4028234663852886e38f, kHighest = 3.4028234663852886e38f;

struct Select {
    size_t sequences, ld;
    int beams, keep, parts;
    unsigned vocabulary, part;      // part: logits, a multiple of kTile
    const void* logits;
    const float* scores;
    const unsigned char* finished;  // or null
    long long end;
    float2* sums;                   // [row][part]: largest logit, sum of exponentials relative to it
    u64* best;                      // [row][part][keep], best first, 0 where there are no more
    float* out_scores;
    long long *out_parents, *out_tokens;
    unsigned char* out_finished;
    size_t first;                   // the launch's first workgroup
};

// A logit as a whole number that orders alike; 0 for what is no candidate.
__device__ __forceinline__ unsigned order_of(float z) {
    const unsigned u = __builtin_bit_cast(unsigned, z);
    return u ^ (unsigned(int(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float logit_of(unsigned o) { return __builtin_bit_cast(float, o ^ (o >> 31 ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ u64 key_of(float z, unsigned place) { return z > -__builtin_inff() ? u64(order_of(z)) << 32 | ~place : 0; }

// A candidate of a sequence: its value as a whole number that orders alike (0: none), and its place among the sequence's.
struct Candidate {
    u64 order, place;
};
__device__ __forceinline__ bool ahead(u64 x, u64 y) { return x > y; }
__device__ __forceinline__ bool ahead(const Candidate& x, const Candidate& y) { return x.order > y.order || (x.order == y.order && x.place < y.place); }
__device__ __forceinline__ u64 better(u64 x, u64 y) { return x > y ? x : y; }
__device__ __forceinline__ Candidate better(const Candidate& x, const Candidate& y) {
    const bool first = ahead(x, y);
    return Candidate{first ? x.order : y.order, first ? x.place : y.place};
}
__device__ __forceinline__ bool exists(u64 x) { return x != 0; }
__device__ __forceinline__ bool exists(const Candidate& x) { return x.order != 0; }

// The `keep` best of `best` (in LDS, best first, none behind the last) and of all threads' v[], no two of which are equal:
// afterwards in `best`.
template <class K, int N> struct Scratch {
    K heads[kThreads + kMaxKeep];
    K list[kMaxKeep * N + kMaxKeep];
    K bound;
    int count;
};
template <class K, int N> __device__ __forceinline__ void take_best(Scratch<K, N>& s, K* best, int keep, const K (&v)[N]) {
    const int tid = threadIdx.x, all = kThreads + keep;
    K own = v[0];
#pragma unroll
    for (int i = 1; i < N; ++i) own = better(own, v[i]);
    __syncthreads();   // (`best` is there, and the last call's readers are done)
    s.heads[tid] = own;
    if (tid < keep) s.heads[kThreads + tid] = best[tid];
    if (tid == 0) { s.bound = K{}; s.count = 0; }
    __syncthreads();
    const auto ranked = [&](const K& key) {
        int rank = 0;
        for (int i = 0; i < all; ++i) rank += ahead(s.heads[i], key);
        if (exists(key) && rank == keep - 1) s.bound = key;
    };
    ranked(own);
    if (tid < keep) ranked(best[tid]);
    __syncthreads();
    const K bound = s.bound;   // at most `keep` threads' heads are not behind it
    const auto offer = [&](const K& key) {
        if (exists(key) && !ahead(bound, key)) s.list[atomicAdd(&s.count, 1)] = key;
    };
    if (!ahead(bound, own))
#pragma unroll
        for (int i = 0; i < N; ++i) offer(v[i]);
    if (tid < keep) offer(best[tid]);
    __syncthreads();
    const int count = s.count;
    if (tid < keep && tid >= count) best[tid] = K{};
    for (int i = tid; i < count; i += kThreads) {
        const K key = s.list[i];
        int rank = 0;
        for (int j = 0; j < count; ++j) rank += ahead(s.list[j], key);
        if (rank < keep) best[rank] = key;
    }
}

template <class Op> __device__ __forceinline__ float all_threads(float v, float* scratch, Op op) {
    v = lanes_fold<kWave>(v, op);
    __syncthreads();   // (the last one's readers are done)
    if (threadIdx.x % kWave == 0) scratch[threadIdx.x / kWave] = v;
    __syncthreads();
    v = scratch[0];
#pragma unroll
    for (int w = 1; w < kThreads / kWave; ++w) v = op(v, scratch[w]);
    return v;
}

template <class T> __global__ __launch_bounds__(kThreads) void part_kernel(Select a) {
    __shared__ Scratch<u64, kVectors * 8> scratch;
    __shared__ u64 best[kMaxKeep];
    __shared__ float waves[kThreads / kWave];
    const size_t block = a.first + blockIdx.x, row = block / unsigned(a.parts);
    const unsigned part = unsigned(block - row * unsigned(a.parts)), begin = part * a.part;
    const unsigned end = a.vocabulary - begin < a.part ? a.vocabulary : begin + a.part;
    if (!(a.scores[row] > -__builtin_inff()) || (a.finished && a.finished[row])) return;   // (its candidates are not read)
    const T* z = static_cast<const T*>(a.logits) + row * a.ld;
    if (int(threadIdx.x) < a.keep) best[threadIdx.x] = 0;
    float most = kLowest, sum = 0.f;
    for (unsigned base = begin; base < end; base += kTile) {
        float8 v[kVectors];
        float m = most;
#pragma unroll
        for (int j = 0; j < kVectors; ++j) {
            const unsigned c = base + (j * kThreads + threadIdx.x) * 8;
            const int n = c < end ? (end - c < 8 ? int(end - c) : 8) : 0;
            v[j] = load8(z + c, n);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[j][i] = i < n && v[j][i] > -__builtin_inff() ? fminf(v[j][i], kHighest) : -__builtin_inff();   // (NaN: minus infinity)
                m = fmaxf(m, v[j][i]);
            }
        }
        sum *= __builtin_amdgcn_exp2f((most - m) * 1.4426950408889634f);
        most = m;
        u64 keys[kVectors * 8];
#pragma unroll
        for (int j = 0; j < kVectors; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                sum += __builtin_amdgcn_exp2f((v[j][i] - most) * 1.4426950408889634f);
                keys[j * 8 + i] = key_of(v[j][i], base + (j * kThreads + threadIdx.x) * 8 + i);
            }
        take_best(scratch, best, a.keep, keys);
    }
    const float m = all_threads(most, waves, [](float x, float y) { return fmaxf(x, y); });
    const float s = all_threads(sum * __builtin_amdgcn_exp2f((most - m) * 1.4426950408889634f), waves, [](float x, float y) { return x + y; });
    if (threadIdx.x == 0) a.sums[block] = float2{m, s};
    if (int(threadIdx.x) < a.keep) a.best[block * a.keep + threadIdx.x] = best[threadIdx.x];
}

__device__ __forceinline__ u64 order_of(double v) {
    const u64 u = __builtin_bit_cast(u64, v);
    return u ^ (u64(static_cast<long long>(u) >> 63) | u64(1) << 63);
}
__device__ __forceinline__ double value_of(u64 o) { return __builtin_bit_cast(double, o ^ (o >> 63 ? u64(1) << 63 : ~u64(0))); }

__global__ __launch_bounds__(kThreads) void join_kernel(Select a) {
    constexpr int kEach = 16;
    __shared__ Scratch<Candidate, kEach> scratch;
    __shared__ Candidate best[kMaxKeep];
    __shared__ double most[kMaxBeams], log_sum[kMaxBeams];
    const size_t sequence = a.first + blockIdx.x, row0 = sequence * a.beams;
    const int tid = threadIdx.x;
    const auto done = [&](int b) { return a.finished && a.finished[row0 + b]; };
    if (tid < a.beams && a.scores[row0 + tid] > -__builtin_inff() && !done(tid)) {
        const float2* sums = a.sums + (row0 + tid) * a.parts;
        float m = kLowest;
        for (int p = 0; p < a.parts; ++p) m = fmaxf(m, sums[p].x);
        double s = 0;
        for (int p = 0; p < a.parts; ++p) s += double(sums[p].y) * exp(double(sums[p].x) - double(m));
        most[tid] = m;
        log_sum[tid] = log(s);
    }
    __syncthreads();
    const int per = a.parts * a.keep, all = a.beams * per;
    const auto candidate = [&](int i) {
        const int b = i / per;
        const float score = a.scores[row0 + b];
        if (!(score > -__builtin_inff())) return Candidate{0, 0};
        if (done(b)) return i == b * per ? Candidate{order_of(double(score)), u64(b) * a.vocabulary + u64(a.end)} : Candidate{0, 0};
        const u64 key = a.best[row0 * per + i];
        if (key == 0) return Candidate{0, 0};
        return Candidate{order_of(double(logit_of(unsigned(key >> 32))) - most[b] - log_sum[b] + double(score)), u64(b) * a.vocabulary + unsigned(~key)};
    };
    if (tid < a.keep) best[tid] = Candidate{0, 0};
    for (int base = 0; base < all; base += kThreads * kEach) {
        Candidate v[kEach];
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int i = base + j * kThreads + tid;
            v[j] = i < all ? candidate(i) : Candidate{0, 0};
        }
        take_best(scratch, best, a.keep, v);
    }
    __syncthreads();
    if (tid >= a.keep) return;
    const Candidate c = best[tid];
    const bool there = exists(c);
    const u64 b = c.place / a.vocabulary;
    const long long token = there ? (long long)(c.place - b * a.vocabulary) : -1;
    const size_t o = sequence * a.keep + tid;
    a.out_scores[o] = there ? float(value_of(c.order)) : -__builtin_inff();
    a.out_parents[o] = there ? (long long)b : tid < a.beams ? tid : 0;
    a.out_tokens[o] = token;
    if (a.out_finished) a.out_finished[o] = token == a.end || token < 0;
}

// ---- the states

constexpr int kMaxStates = 16;
struct State {
    char* data;
    size_t stride, bytes;
    unsigned slabs;      // workgroups a sequence
    size_t first;        // its first workgroup
};
struct Reorder {
    const long long* parents;
    int beams, count;
    State states[kMaxStates];
};

template <class V> __device__ __forceinline__ V load_any(const char* p) {
    V v;
    __builtin_memcpy(&v, __builtin_assume_aligned(p, 1), sizeof(v));
    return v;
}

// A thread reads its 16 bytes of all beams that move before it writes any, so that nothing is in another's way.
template <int B> __global__ __launch_bounds__(kThreads) void reorder_kernel(Reorder a) {
    int i = 0;
    while (i + 1 < a.count && a.states[i + 1].first <= blockIdx.x) ++i;
    const State& s = a.states[i];
    const size_t block = blockIdx.x - s.first, sequence = block / s.slabs;
    const size_t at = ((block - sequence * s.slabs) * kThreads + threadIdx.x) * 16;
    const long long* parents = a.parents + sequence * a.beams;
    int from[B];
#pragma unroll
    for (int b = 0; b < B; ++b) {
        const long long p = b < a.beams ? parents[b] : b;
        from[b] = p >= 0 && p < a.beams ? int(p) : b;
    }
    if (at >= s.bytes) return;
    char* row = s.data + sequence * a.beams * s.stride + at;
    if (s.bytes - at >= 16) {
        floatx4 v[B];
#pragma unroll
        for (int b = 0; b < B; ++b)
            if (from[b] != b) v[b] = load_any<floatx4>(row + from[b] * s.stride);
#pragma unroll
        for (int b = 0; b < B; ++b)
            if (from[b] != b) __builtin_memcpy(__builtin_assume_aligned(row + b * s.stride, 1), &v[b], 16);
    } else {
        for (size_t j = 0; j < s.bytes - at; ++j) {
            char v[B];
#pragma unroll
            for (int b = 0; b < B; ++b)
                if (from[b] != b) v[b] = row[from[b] * s.stride + j];
#pragma unroll
            for (int b = 0; b < B; ++b)
                if (from[b] != b) row[b * s.stride + j] = v[b];
        }
    }
}

// ---- host side

constexpr size_t kMostBlocks = 0xffffffffu / kThreads;

bool valid(const flstm_beams* p) {
    return p && valid_dtype(p->dtype) && p->sequences < (size_t(1) << 31) && p->beams >= 1 && p->beams <= kMaxBeams && p->keep >= 1 &&
           p->keep <= kMaxKeep && p->vocabulary >= 1 && p->vocabulary < (size_t(1) << 31) - 65536 && p->ld >= p->vocabulary &&
           (!p->finished || (p->end >= 0 && p->end < (long long)p->vocabulary)) && (p->sequences == 0 || (p->logits && p->scores));
}
size_t part_of(const flstm_beams* p) { return round_up(ceil_div(p->vocabulary, kMaxParts), kTile); }
size_t parts_of(const flstm_beams* p) { return ceil_div(p->vocabulary, part_of(p)); }
size_t best_bytes(const flstm_beams* p) { return round_up(p->sequences * p->beams * parts_of(p) * p->keep * sizeof(u64), 16); }

}  // namespace
}  // namespace flstm_hip

using namespace flstm_hip;

extern "C" size_t flstm_beam_select_workspace_bytes(const flstm_beams* p) {
    return valid(p) ? best_bytes(p) + p->sequences * p->beams * parts_of(p) * sizeof(float2) : 0;
}

extern "C" int flstm_beam_select(const flstm_beams* p, float* scores, long long* parents, long long* tokens, unsigned char* finished, void* workspace,
                                 void* stream) {
    if (!valid(p)) return FLSTM_E_INVALID;
    if (p->sequences == 0) return 0;
    if (!scores || !parents || !tokens || !workspace) return FLSTM_E_INVALID;
    Select a{};
    a.sequences = p->sequences; a.ld = p->ld; a.beams = p->beams; a.keep = p->keep; a.vocabulary = unsigned(p->vocabulary);
    a.part = unsigned(part_of(p)); a.parts = int(parts_of(p)); a.logits = p->logits; a.scores = p->scores; a.finished = p->finished;
    a.end = p->end; a.best = static_cast<u64*>(workspace); a.sums = reinterpret_cast<float2*>(static_cast<char*>(workspace) + best_bytes(p));
    a.out_scores = scores; a.out_parents = parents; a.out_tokens = tokens; a.out_finished = finished;
    const size_t blocks = p->sequences * p->beams * a.parts;
    hipStream_t s = static_cast<hipStream_t>(stream);
    for (a.first = 0; a.first < blocks; a.first += kMostBlocks) {
        const unsigned some = unsigned(blocks - a.first < kMostBlocks ? blocks - a.first : kMostBlocks);
        const int rc = with_type(p->dtype, [&](auto zero) {
            part_kernel<decltype(zero)><<<some, kThreads, 0, s>>>(a);
            return launched();
        });
        if (rc != 0) return rc;
    }
    for (a.first = 0; a.first < p->sequences; a.first += kMostBlocks) {
        join_kernel<<<unsigned(p->sequences - a.first < kMostBlocks ? p->sequences - a.first : kMostBlocks), kThreads, 0, s>>>(a);
        if (const int rc = launched()) return rc;
    }
    return 0;
}

extern "C" int flstm_beam_reorder(size_t sequences, int beams, const long long* parents, const flstm_beam_state* states, int count, void* stream) {
    if (beams < 1 || beams > kMaxBeams || count < 0 || count > kMaxStates || (count > 0 && !states)) return FLSTM_E_INVALID;
    if (sequences == 0 || count == 0 || beams == 1) return 0;
    if (!parents) return FLSTM_E_INVALID;
    Reorder a{};
    a.parents = parents; a.beams = beams;
    size_t blocks = 0;
    for (int i = 0; i < count; ++i) {
        if (states[i].bytes == 0) continue;
        if (!states[i].data || states[i].stride < states[i].bytes) return FLSTM_E_INVALID;
        const size_t slabs = ceil_div(states[i].bytes, kThreads * 16);
        if (slabs > kMostBlocks || sequences > kMostBlocks / slabs) return FLSTM_E_TOO_LARGE;
        a.states[a.count++] = State{static_cast<char*>(states[i].data), states[i].stride, states[i].bytes, unsigned(slabs), blocks};
        blocks += slabs * sequences;
    }
    if (blocks > kMostBlocks) return FLSTM_E_TOO_LARGE;
    if (blocks == 0) return 0;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (beams <= 4) reorder_kernel<4><<<unsigned(blocks), kThreads, 0, s>>>(a);
    else if (beams <= 8) reorder_kernel<8><<<unsigned(blocks), kThreads, 0, s>>>(a);
    else if (beams <= 16) reorder_kernel<16><<<unsigned(blocks), kThreads, 0, s>>>(a);
    else reorder_kernel<32><<<unsigned(blocks), kThreads, 0, s>>>(a);
    return launched();
}
