// Beam search (lm_ops.h): the best continuations of every sequence's beams, and the beams' states moved behind them.
//
// The selection is bound by one reading of the logits.  A workgroup has a part of a row: the part's largest logit, the sum of its
// exponentials, and its `keep` best entries, all from registers.  Its threads form at least `keep` groups; the smallest of the
// groups' largest logits is a bound that `keep` entries reach and few others do (20 of 8192 random ones for 8, 110 for 32), so that what
// is ordered is a short list.  Ordered are whole numbers, the logit's order above and the place's complement below: no two are equal,
// and equal logits come lowest place first.  Of very many logits that are equal to the bound the lowest
// places are listed, bounded the same way; where even that is too long, the best are taken out one by one.  A second kernel puts the parts together: the rows' logarithms, and the continuations' values in 64
// bits, so that which of a row's is larger does not depend on a rounding to 32.  The logarithm is that of a sum in 32 bits, off by up to 48 units of 2^-24: values of
// different rows that are nearer to each other may come in either order, those of equal rows and scores come lowest first.
// 512 rows of 50001 bf16 logits, 8 of each sequence's 8 kept: 17.0 us for the parts, 3.0 TB/s at four fifths of the vector units, and 7.6 for putting them
// together, a chain of trips to memory and through LDS.  The states move at what memory gives: 137 MB in 22 us.
#include "lm_device.h"

namespace flstm_hip {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxKeep = 32, kMaxBeams = 32;
constexpr int kVectors = 4, kTile = kThreads * kVectors * 8;   // logits a workgroup holds at a time
constexpr size_t kMaxParts = 64;   // one for each lane of a wave
constexpr int kList = 1024;        // entries that are ordered at once
static_assert(kTile <= kList * 8);
constexpr float kLog2e = 1.4426950408889634f, kLowest = -3.4028234663852886e38f, kHighest = 3.4028234663852886e38f;

struct Select {
    size_t sequences, ld;
    int beams, keep, parts;
    unsigned vocabulary, part;      // part: logits
    int groups;                     // of threads, 4 to 32, a power of two, no fewer than `keep`
    const void* logits;
    const float* scores;
    const unsigned char* finished;  // or null
    long long end;
    float2* sums;                   // [row][part]: largest logit, sum of exponentials relative to it
    u64* best;                      // [row][part][keep], best first, 0 where there are no more
    float* out_scores;
    long long *out_parents, *out_tokens;
    unsigned char* out_finished;
    size_t first;                   // the launch's first row, or sequence
};

// A logit as a whole number that orders alike, zeros of either sign the same; 0 for what is no candidate.
__device__ __forceinline__ unsigned order_of(float z) {
    const unsigned u = __builtin_bit_cast(unsigned, z + 0.f);   // (-0 + 0 is +0)
    return u ^ (unsigned(int(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float logit_of(unsigned o) { return __builtin_bit_cast(float, o ^ (o >> 31 ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ u64 key_of(float z, unsigned place) { return z > -__builtin_inff() ? u64(order_of(z)) << 32 | ~place : 0; }

// A value folded over the lanes l, l + groups, l + 2 groups, .. of a wave.
template <class Op> __device__ __forceinline__ float groups_fold(float v, int groups, Op op) {
    unsigned u = __builtin_bit_cast(unsigned, v);
    const auto across = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    v = op(__builtin_bit_cast(float, unsigned(across[0])), __builtin_bit_cast(float, unsigned(across[1])));
    if (groups <= 16) {
        u = __builtin_bit_cast(unsigned, v);
        const auto rows = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        v = op(__builtin_bit_cast(float, unsigned(rows[0])), __builtin_bit_cast(float, unsigned(rows[1])));
    }
    if (groups <= 8) v = op(v, lane_moved<0x128>(v));   // row_ror 8
    if (groups <= 4) v = op(v, lane_moved<0x124>(v));   // row_ror 4
    return v;
}

// A logit as a number: minus infinity for a NaN, the largest finite one for infinity.
__device__ __forceinline__ float number(float x) { return x > -__builtin_inff() ? fminf(x, kHighest) : -__builtin_inff(); }

// The largest of the workgroup's, in all threads.
__device__ __forceinline__ u64 all_largest(u64 v, u64* scratch) {
#pragma unroll
    for (int d = kWave / 2; d > 0; d /= 2) {
        const u64 other = __shfl_xor(v, d);
        v = other > v ? other : v;
    }
    __syncthreads();
    if (threadIdx.x % kWave == 0) scratch[threadIdx.x / kWave] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / kWave; ++w) v = scratch[w] > v ? scratch[w] : v;
    return v;
}

// The list again where very many logits are equal to the bound (those that a mask left at its type's lowest value, say): of these, those up to
// a place that the first ones of all groups reach.  Returns how many there are then.
template <class T> __device__ int fewer(const T* z, unsigned base, unsigned end, float bound, int groups, unsigned* places, float (*heads)[kMaxKeep], int& count) {
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    const unsigned stop = end - base < unsigned(kTile) ? end - base : kTile;
    float first = __builtin_inff();
    for (unsigned c = tid; c < stop; c += kThreads) {
        const float x = number(float(z[base + c]));
        if (x >= bound) first = fminf(first, x > bound ? -1.f : float(c));   // (a group with one above it needs no equal one)
    }
    first = groups_fold(first, groups, [](float x, float y) { return fminf(x, y); });
    __syncthreads();   // (the readers of `count` and `heads` are done)
    if (lane < groups) heads[wave][lane] = first;
    if (tid == 0) count = 0;
    __syncthreads();
    first = heads[0][lane % groups];
    for (int w = 1; w < kThreads / kWave; ++w) first = fminf(first, heads[w][lane % groups]);
    const float place = lanes_max<kWave>(first);
    for (unsigned c = tid; c < stop; c += kThreads) {
        const float x = number(float(z[base + c]));
        if (x > bound || (x == bound && float(c) <= place)) {
            const int at = atomicAdd(&count, 1);
            if (at < kList) places[at] = base + c;
        }
    }
    __syncthreads();
    return count;
}

template <class T> __global__ __launch_bounds__(kThreads) void part_kernel(Select a) {
    __shared__ u64 list[kList + kMaxKeep], best[kMaxKeep], largest[kThreads / kWave];
    __shared__ unsigned places[kList];   // no fewer than a tile's vectors
    __shared__ float heads[kThreads / kWave][kMaxKeep], waves[kThreads / kWave];
    __shared__ int count, vectors;   // entries and vectors that reach the bound
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    const unsigned in_launch = blockIdx.x / unsigned(a.parts), part = blockIdx.x - in_launch * unsigned(a.parts), begin = part * a.part;
    const size_t row = a.first + in_launch, block = row * unsigned(a.parts) + part;
    const unsigned end = a.vocabulary - begin < a.part ? a.vocabulary : begin + a.part;
    if (!(a.scores[row] > -__builtin_inff()) || (a.finished && a.finished[row])) return;   // (its continuations are not read)
    const T* z = static_cast<const T*>(a.logits) + row * a.ld;
    float most = kLowest, sum = 0.f;
    for (unsigned base = begin; base < end; base += kTile) {
        typename Vec8<T>::type v[kVectors];   // as they come: converted three times, in half the registers
        float m = -__builtin_inff();
        const auto place_of = [&](int j) {   // of a vector's first entry
            const unsigned c = base + (j * kThreads + tid) * 8;
            return c + 8 > end && a.vocabulary >= 8 ? end - 8 : c;
        };
        // All vectors are requested without a branch, behind which they would be waited for one by one: the last one of the part from where it ends, and what is
        // not this thread's of it taken out.  (Rows of less than a vector: piece by piece.)
        if (a.vocabulary >= 8) {
#pragma unroll
            for (int j = 0; j < kVectors; ++j) {
                __builtin_memcpy(&v[j], __builtin_assume_aligned(z + place_of(j), sizeof(T)), sizeof(v[j]));
            }
#pragma unroll
            for (int j = 0; j < kVectors; ++j) {
                const unsigned c = base + (j * kThreads + tid) * 8;
                if (c + 8 > end)
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[j][i] = c < end && place_of(j) + i >= c ? v[j][i] : T(-__builtin_inff());
            }
        } else {
#pragma unroll
            for (int j = 0; j < kVectors; ++j) v[j] = T(-__builtin_inff());
            if (tid == 0)
#pragma unroll
                for (int i = 0; i < 8; ++i) v[0][i] = unsigned(i) < end ? z[i] : v[0][i];
        }
#pragma unroll
        for (int j = 0; j < kVectors; ++j) {
            asm volatile("" : "+v"(v[j]));
#pragma unroll
            for (int i = 0; i < 8; ++i) m = fmaxf(m, float(v[j][i]));   // (a NaN is no one's maximum)
        }
        m = groups_fold(fminf(m, kHighest), a.groups, [](float x, float y) { return fmaxf(x, y); });
        if (lane < a.groups) heads[wave][lane] = m;
        if (tid == 0) count = vectors = 0;
        __syncthreads();
        m = heads[0][lane % a.groups];
#pragma unroll
        for (int w = 1; w < kThreads / kWave; ++w) m = fmaxf(m, heads[w][lane % a.groups]);
        float bound = lanes_fold<kWave>(m, [](float x, float y) { return fminf(x, y); });
        bound = fmaxf(bound, kLowest);   // (minus infinity is no continuation)
        if (base > begin && best[a.keep - 1]) bound = fmaxf(bound, logit_of(unsigned(best[a.keep - 1] >> 32)));
        m = fmaxf(most, lanes_max<kWave>(m));
        sum *= __builtin_amdgcn_exp2f((most - m) * kLog2e);
        most = m;
        // exponents as one operation each, z log2(e) - shift; what the rounding of shift is off by is put right behind the sum, as long as that leaves the sum's terms in
        // range (most below 2^30, say: beyond it a step of shift can be a factor of 2^64 and more)
        const float shift = most * kLog2e, off = __builtin_fmaf(most, kLog2e, -shift);
        const float reached = __builtin_fmaf(bound, kLog2e, -shift);   // (rounding keeps the order)
        float more = 0.f;
        unsigned reach = 0;   // a bit for each of this thread's vectors: whether an entry reaches the bound
#pragma unroll
        for (int j = 0; j < kVectors; ++j) {
            asm volatile("" : "+v"(v[j]));
            float largest_d = -__builtin_inff();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float d = __builtin_fmaf(float(v[j][i]), kLog2e, -shift);
                more += __builtin_amdgcn_exp2f(d);
                largest_d = fmaxf(largest_d, d);
            }
            reach |= largest_d < reached ? 0u : 1u << j;
        }
        while (reach) {
            const int j = __ffs(int(reach)) - 1;
            reach &= reach - 1;
            places[atomicAdd(&vectors, 1)] = base + (j * kThreads + tid) * 8;
        }
        if (more < __builtin_inff() && fabsf(off) <= 64.f) {
            more *= __builtin_amdgcn_exp2f(-off);
        } else {   // a NaN or an infinity among them, or exponents that are none: once more, number by number
            more = 0.f;
            for (int i = 0; i < kVectors * 8; ++i) {
                const unsigned c = base + (i / 8 * kThreads + tid) * 8 + i % 8;
                if (c < end) more += __builtin_amdgcn_exp2f((number(float(z[c])) - most) * kLog2e);
            }
        }
        sum += more;
        if (base + kTile >= end) {
            sum = lanes_sum<kWave>(sum);
            if (lane == 0) waves[wave] = sum;
        }
        const u64 before = base > begin && tid < a.keep ? best[tid] : 0;   // of the tiles in front
        __syncthreads();
        // which of the vectors' entries do: looked up again, a lane each, for fewer instructions than keeping account of all
        for (int i = tid; i < vectors * 8; i += kThreads) {
            const unsigned c = places[i / 8] + i % 8;
            if (c >= end) continue;
            const float x = number(float(z[c]));
            if (!(x >= bound)) continue;
            const int at = atomicAdd(&count, 1);
            if (at < kList) list[at] = key_of(x, c);
        }
        __syncthreads();
        int some = count;
        if (some > kList) {
            some = fewer(z, base, end, bound, a.groups, places, heads, count);
            if (some <= kList)
                for (int i = tid; i < some; i += kThreads) list[i] = key_of(number(float(z[places[i]])), places[i]);
        }
        if (some <= kList) {
            if (base > begin) {
                if (tid < a.keep) list[some + tid] = before;
                some += a.keep;
            }
            if (tid < a.keep) best[tid] = 0;
            __syncthreads();
            for (int i = tid; i < some; i += kThreads) {
                const u64 key = list[i];
                int rank = 0;
#pragma unroll 8
                for (int j = 0; j < some; ++j) rank += list[j] > key;
                if (rank < a.keep && key) best[rank] = key;
            }
        } else {
            u64 last = ~u64(0);
            for (int r = 0; r < a.keep; ++r) {
                u64 key = before < last ? before : 0;
                for (unsigned c = base + tid; c < end && c < base + kTile; c += kThreads) {
                    const u64 k = key_of(number(float(z[c])), c);
                    key = k < last && k > key ? k : key;
                }
                last = all_largest(key, largest);
                if (tid == 0) best[r] = last;
            }
        }
        __syncthreads();
    }
    if (tid == 0) {
        float s = waves[0];
#pragma unroll
        for (int w = 1; w < kThreads / kWave; ++w) s += waves[w];
        a.sums[block] = float2{most, s};
    }
    if (tid < a.keep) a.best[block * a.keep + tid] = best[tid];
}

// A continuation of a sequence: its value as a whole number that orders alike (0: none), and its place among the sequence's.
struct Candidate {
    u64 order, place;
};
__device__ __forceinline__ bool ahead(const Candidate& x, const Candidate& y) { return x.order > y.order || (x.order == y.order && x.place < y.place); }
__device__ __forceinline__ u64 order_of(double v) {
    const u64 u = __builtin_bit_cast(u64, v + 0.);
    return u ^ (u64(static_cast<long long>(u) >> 63) | u64(1) << 63);
}
__device__ __forceinline__ double value_of(u64 o) { return __builtin_bit_cast(double, o ^ (o >> 63 ? u64(1) << 63 : ~u64(0))); }

__global__ __launch_bounds__(kThreads) void join_kernel(Select a) {
    __shared__ Candidate list[kList], best[kMaxKeep];
    __shared__ u64 heads[kThreads / kWave][kMaxKeep], largest[kThreads / kWave];
    __shared__ double most[kMaxBeams], rest[kMaxBeams];   // a row's largest logit; what its difference to one is off by
    __shared__ int state[kMaxBeams];        // of a hypothesis: 0 none, 1 alive, 2 finished
    __shared__ int count;
    const size_t sequence = a.first + blockIdx.x, row0 = sequence * a.beams;
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    // The best of all parts first, then the second, and so on: so each group of threads has some of the first, and its bound is close where parts are
    // alike.  Where a part holds all of the best, the last of its entries is one that is closer; the larger of the two counts.
    const int lists = a.beams * a.parts, all = lists * a.keep;
    const float by_lists = 1.f / float(lists), by_parts = 1.f / float(a.parts);
    const auto quotient = [](int i, float inverse) { return int((float(i) + 0.5f) * inverse); };   // (of numbers below 2^17: half a step is more than any error)
    const auto key_at = [&](int i) {
        const int rank = quotient(i, by_lists);
        return a.best[(row0 * a.parts + (i - rank * lists)) * a.keep + rank];
    };
    constexpr int kHeld = 8;   // of a thread's continuations, requested at once
    u64 held[kHeld];
#pragma unroll
    for (int j = 0; j < kHeld; ++j) held[j] = tid + j * kThreads < all ? key_at(tid + j * kThreads) : 0;
    for (int b = wave; b < a.beams; b += kThreads / kWave) {
        const float score = a.scores[row0 + b];
        const bool done = a.finished && a.finished[row0 + b], alive = score > -__builtin_inff() && !done;
        float2 p{kLowest, 0.f};
        if (alive && lane < a.parts) p = a.sums[(row0 + b) * a.parts + lane];
        const float m = lanes_max<kWave>(p.x), s = lanes_sum<kWave>(p.y * __builtin_amdgcn_exp2f((p.x - m) * kLog2e));
        if (lane == 0) {
            most[b] = m;
            rest[b] = done ? double(score) : double(score) - log(double(s));
            state[b] = !(score > -__builtin_inff()) ? 0 : done ? 2 : 1;
        }
    }
    if (tid < a.keep) best[tid] = Candidate{0, 0};
    if (tid == 0) count = 0;
    __syncthreads();
    const auto candidate_of = [&](int i, u64 key) {
        const int rank = quotient(i, by_lists), b = quotient(i - rank * lists, by_parts);
        const u64 row = u64(b) * a.vocabulary;
        if (state[b] == 2) return i == b * a.parts ? Candidate{order_of(rest[b]), row + u64(a.end)} : Candidate{0, 0};
        return key && state[b] == 1 ? Candidate{order_of(double(logit_of(unsigned(key >> 32))) - most[b] + rest[b]), row + unsigned(~key)} : Candidate{0, 0};
    };
    const auto candidate = [&](int i) { return candidate_of(i, key_at(i)); };
    u64 head = 0, end_of_list = 0, orders[kHeld];
    const auto heads_of = [&](int i, u64 o) {
        head = o > head ? o : head;
        if (i >= all - lists) end_of_list = o > end_of_list ? o : end_of_list;
    };
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
        const int i = tid + j * kThreads;
        orders[j] = i < all ? candidate_of(i, held[j]).order : 0;
        heads_of(i, orders[j]);
    }
    for (int i = tid + kHeld * kThreads; i < all; i += kThreads) heads_of(i, candidate(i).order);
#pragma unroll
    for (int d = kWave / 2; d > 0; d /= 2) {
        const u64 other = __shfl_xor(end_of_list, d);
        end_of_list = other > end_of_list ? other : end_of_list;
    }
    if (lane == 0) largest[wave] = end_of_list;
    for (int d = kWave / 2; d >= a.groups; d /= 2) {
        const u64 other = __shfl_xor(head, d);
        head = other > head ? other : head;
    }
    if (lane < a.groups) heads[wave][lane] = head;
    __syncthreads();
    u64 bound = heads[0][lane % a.groups];
#pragma unroll
    for (int w = 1; w < kThreads / kWave; ++w) bound = heads[w][lane % a.groups] > bound ? heads[w][lane % a.groups] : bound;
    for (int d = a.groups / 2; d > 0; d /= 2) {
        const u64 other = __shfl_xor(bound, d);
        bound = other < bound ? other : bound;
    }
#pragma unroll
    for (int w = 0; w < kThreads / kWave; ++w) bound = largest[w] > bound ? largest[w] : bound;
    const auto offer = [&](const Candidate& c) {
        if (c.order && c.order >= bound) {
            const int at = atomicAdd(&count, 1);
            if (at < kList) list[at] = c;
        }
    };
#pragma unroll
    for (int j = 0; j < kHeld; ++j)
        if (orders[j] && orders[j] >= bound) offer(candidate_of(tid + j * kThreads, held[j]));
    for (int i = tid + kHeld * kThreads; i < all; i += kThreads) offer(candidate(i));
    __syncthreads();
    const int some = count;
    if (some <= kList) {
        for (int i = tid; i < some; i += kThreads) {
            const Candidate c = list[i];
            int rank = 0;
#pragma unroll 8
            for (int j = 0; j < some; ++j) rank += ahead(list[j], c);
            if (rank < a.keep) best[rank] = c;
        }
    } else {
        u64 last = ~u64(0), last_place = 0;
        for (int r = 0; r < a.keep; ++r) {   // the largest value behind the last one, and the lowest place that has it
            u64 o = 0, place = ~u64(0);
            for (int i = tid; i < all; i += kThreads) {
                const Candidate c = candidate(i);
                if (c.order && (c.order < last || (c.order == last && c.place > last_place)) && (c.order > o || (c.order == o && c.place < place))) {
                    o = c.order;
                    place = c.place;
                }
            }
            last = all_largest(o, largest);
            last_place = ~all_largest(o == last ? ~place : 0, largest);
            if (tid == 0 && last) best[r] = Candidate{last, last_place};
            if (!last) break;
        }
    }
    __syncthreads();
    if (tid >= a.keep) return;
    const Candidate c = best[tid];
    const bool there = c.order != 0;
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
    unsigned first;      // its first workgroup
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
    const unsigned block = blockIdx.x - s.first, sequence = block / s.slabs;
    const size_t at = (size_t(block - sequence * s.slabs) * kThreads + threadIdx.x) * 16;
    const long long* parents = a.parents + size_t(sequence) * a.beams;
    int from[B];
#pragma unroll
    for (int b = 0; b < B; ++b) {
        const long long p = b < a.beams ? parents[b] : b;
        from[b] = p >= 0 && p < a.beams ? int(p) : b;
    }
    if (at >= s.bytes) return;
    char* row = s.data + size_t(sequence) * a.beams * s.stride + at;
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

// `count` rows of `bytes` at every `stride` from `at` on; whether two such have memory in common, where one launch would move it twice.  Rows may lie between
// each other's (halves of a wider state).
struct Extent {
    size_t at, stride, bytes, count;
};
bool meet(Extent x, Extent y) {
    if (y.at < x.at) {
        const Extent z = x;
        x = y;
        y = z;
    }
    const size_t apart = y.at - x.at;
    if (apart / x.stride >= x.count || (apart / x.stride == x.count - 1 && apart % x.stride >= x.bytes)) return false;
    if (x.stride == y.stride) return apart % x.stride < x.bytes || x.stride - apart % x.stride < y.bytes;
    for (size_t i = apart / x.stride, j = 0; i < x.count && j < y.count;) {   // a row each, of which the one in front does not reach the other
        const size_t of_x = i * x.stride, of_y = apart + j * y.stride;
        if (of_x <= of_y ? of_y - of_x < x.bytes : of_x - of_y < y.bytes) return true;
        if (of_x <= of_y) i = of_y / x.stride > i ? of_y / x.stride : i + 1;
        else j = (of_x - apart) / y.stride > j ? (of_x - apart) / y.stride : j + 1;
    }
    return false;
}

constexpr size_t kMostBlocks = 0xffffffffu / kThreads;

bool valid(const flstm_beams* p) {
    return p && valid_dtype(p->dtype) && p->sequences < (size_t(1) << 31) && p->beams >= 1 && p->beams <= kMaxBeams && p->keep >= 1 &&
           p->keep <= kMaxKeep && p->vocabulary >= 1 && p->vocabulary < (size_t(1) << 31) - 65536 && p->ld >= p->vocabulary &&
           (!p->finished || (p->end >= 0 && p->end < (long long)p->vocabulary)) && (p->sequences == 0 || (p->logits && p->scores));
}
// Rows in parts of about one size, none above kTile as long as kMaxParts are enough.
size_t part_of(const flstm_beams* p) {
    const size_t parts = ceil_div(p->vocabulary, kTile);
    return round_up(ceil_div(p->vocabulary, parts < kMaxParts ? parts : kMaxParts), 64);
}
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
    a.groups = 4;
    while (a.groups < a.keep) a.groups *= 2;
    a.end = p->end; a.best = static_cast<u64*>(workspace); a.sums = reinterpret_cast<float2*>(static_cast<char*>(workspace) + best_bytes(p));
    a.out_scores = scores; a.out_parents = parents; a.out_tokens = tokens; a.out_finished = finished;
    const size_t rows = p->sequences * p->beams, most = kMostBlocks / a.parts;   // rows a launch
    hipStream_t s = static_cast<hipStream_t>(stream);
    for (a.first = 0; a.first < rows; a.first += most) {
        const unsigned some = unsigned((rows - a.first < most ? rows - a.first : most) * a.parts);
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
    if (beams < 1 || beams > kMaxBeams || count < 0 || (count > 0 && !states)) return FLSTM_E_INVALID;
    if (sequences == 0 || count == 0 || beams == 1) return 0;
    if (!parents) return FLSTM_E_INVALID;
    if (sequences > ~size_t(0) / kMaxBeams) return FLSTM_E_TOO_LARGE;
    const Extent index{reinterpret_cast<size_t>(parents), sizeof(*parents), sizeof(*parents), sequences * beams};
    const auto extent = [&](int i) { return Extent{reinterpret_cast<size_t>(states[i].data), states[i].stride, states[i].bytes, sequences * beams}; };
    const auto slabs = [&](int i) { return ceil_div(states[i].bytes, kThreads * 16); };
    for (int i = 0; i < count; ++i) {
        if (states[i].bytes == 0) continue;
        if (!states[i].data || states[i].stride < states[i].bytes) return FLSTM_E_INVALID;
        if (slabs(i) > kMostBlocks / sequences) return FLSTM_E_TOO_LARGE;
        if (meet(index, extent(i))) return FLSTM_E_INVALID;
        for (int j = 0; j < i; ++j)
            if (states[j].bytes && meet(extent(j), extent(i))) return FLSTM_E_INVALID;
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    for (int i = 0; i < count;) {
        Reorder a{};
        a.parents = parents; a.beams = beams;
        size_t blocks = 0;
        for (; i < count && a.count < kMaxStates && blocks + slabs(i) * sequences <= kMostBlocks; ++i) {
            if (states[i].bytes == 0) continue;
            a.states[a.count++] = State{static_cast<char*>(states[i].data), states[i].stride, states[i].bytes, unsigned(slabs(i)), unsigned(blocks)};
            blocks += slabs(i) * sequences;
        }
        if (blocks == 0) break;
        if (beams <= 4) reorder_kernel<4><<<unsigned(blocks), kThreads, 0, s>>>(a);
        else if (beams <= 8) reorder_kernel<8><<<unsigned(blocks), kThreads, 0, s>>>(a);
        else if (beams <= 16) reorder_kernel<16><<<unsigned(blocks), kThreads, 0, s>>>(a);
        else reorder_kernel<32><<<unsigned(blocks), kThreads, 0, s>>>(a);
        if (const int rc = launched()) return rc;
    }
    return 0;
}
