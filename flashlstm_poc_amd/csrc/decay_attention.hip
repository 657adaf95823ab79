// Attention with a decaying state (lm_ops.h): prompts and training in chunks of tokens, single tokens by themselves.
//
// One sweep serves the forward pass and all three gradients.  For rows q, k (D wide) and v (E wide) it walks the tokens with a
// D x E state X and a decay g:
//     out_t = a g q_t X_{t-1} + b sum_{s in t's chunk, s <= t} g^(t-s) (q_t . k_s) v_s,   X_t = g X_{t-1} + c k_t v_t^T
// Forward it is called with (q, k, v).  With A_s = scale q_s do_s^T + g A_{s+1} the gradients are
//     dq_t = scale S_t do_t:  the sweep of (do, v, k) with the transposed state;
//     dv_s = A_s^T k_s, dk_s = A_s v_s:  the sweeps of (k, q, do) and (v, do, q) from the last token to the first.
//
// A workgroup holds X of one head (128 columns of it at most) in its accumulators for a whole run of tokens, so that a token's rows
// are read once, its output written once, and nothing else leaves the chip.  Each wave has 32 columns of X and forms the scores of
// a chunk for itself: four times these products, and no exchange.  (Shared out through LDS, in tiles of 16 x 16 and with a third
// barrier a chunk, they took the same time for heads of 128, 13 to 17 % more for heads of 64 and 6 % less for fp32, while the outputs'
// operands were in one part.)  The layouts
// are chosen so that no accumulator passes through LDS: in every product below the operand that was an accumulator before has its
// contraction index where the accumulator rows lie (see `perm`).
//
// What bounds it is the chain of a chunk, not one unit: the next rows are requested under the products, written to LDS between two
// barriers, multiplied, weighted, multiplied again.  A workgroup alone on its CU takes 10400 clocks for a chunk of 64 tokens of a
// head of 128 x 128 (barrier and the rows' arrival 640, staging 1350, products with rows and state 2670, weights and outputs 2960,
// requests 600, the state 2220; 3700 of them MFMA), each of two 13900.  Kernels alone, under the profiler, bf16 but for the second: 16 x 2048
// tokens of 16 heads of 128 forward 209 us (2.6 TB/s of rows), their gradients 467; 131072 tokens of 8 heads, fp16, 143 for what segments
// add, 15, and 338; a copy reaches 5.1 TB/s.  fp32: the matrix units are busy for 55 % of the forward pass (16 x 512 tokens of 16 heads,
// 184 us) and 65 % of the gradients' (8192 tokens of 8 heads, 220 us); a third of that is scores, which each wave forms for itself.
#include "lm_device.h"

namespace flstm_hip {
namespace {

constexpr int kMinHead = 8, kMaxHead = 256;     // dk, dv (8: a 16-byte slot of the narrower types)

typedef unsigned uint4v __attribute__((ext_vector_type(4)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4v lds_short4;

// Tokens a chunk: fp32 tiles are twice as large.
template <class T> constexpr int kChunk = sizeof(T) == 4 ? 32 : 64;

// Rows of one role: element (n, t, h, i) at data + n * sequence + t * token + (h / group) * head + i.
struct Role {
    void* data;
    ptrdiff_t sequence, token, head;
    int group;
};

struct Sweep {
    Role q, k, v, out;
    int d, e;              // widths of (q, k) and (v, out)
    int out_f32;           // out holds floats whatever the type (shares of heads that are summed afterwards)
    int reverse;           // from the last token to the first; x_in then belongs to the last token itself
    const float* x_in;     // null: zeros
    float* x_out;          // null: not written
    int in_d, in_e, out_d, out_e;         // strides of a state's elements; states lie d * e apart
    int in_slots, out_slots;              // states are counted by segment, not by sequence
    float a, b, c;
};

struct Sweeps {
    Sweep s[3];
    int count;
    size_t sequences, tokens, slots, segment;   // segment: tokens a workgroup walks at most, a multiple of every chunk
    const int* cu_seqlens;
    int heads, column_blocks;
    const float* log_decay;
};

// The tokens of sequence n, whatever cu_seqlens holds; n == sequences: those behind the last.
struct Span { long long first, length; };
__device__ __forceinline__ Span span_of(const Sweeps& a, long long n) {
    if (!a.cu_seqlens) return Span{0, (long long)a.tokens};
    const long long all = (long long)a.tokens;
    const auto bound = [&](long long i) {
        if (i <= 0) return 0ll;
        if (i > (long long)a.sequences) return all;
        const long long v = a.cu_seqlens[i];
        return v < 0 ? 0ll : v > all ? all : v;
    };
    const long long first = bound(n), end = bound(n + 1);
    return Span{first, end > first ? end - first : 0};
}
// A sequence's segments have consecutive slots.  Packed: from first / segment + n on, which leaves each enough of them without
// a sum over the sequences before.
__device__ __forceinline__ long long first_slot(const Sweeps& a, long long n) {
    if (!a.cu_seqlens) return n * (long long)(a.tokens ? (a.tokens + a.segment - 1) / a.segment : 1);
    return span_of(a, n).first / (long long)a.segment + n;
}
__device__ __forceinline__ long long sequence_of(const Sweeps& a, long long slot) {
    if (!a.cu_seqlens) return slot / (long long)(a.tokens ? (a.tokens + a.segment - 1) / a.segment : 1);
    long long lo = 0, hi = (long long)a.sequences;   // the last n whose first slot is not behind this one
    while (lo < hi) {
        const long long mid = (lo + hi + 1) / 2;
        if (first_slot(a, mid) <= slot) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// exp2(n * l), 1 for n == 0 also where l is minus infinity.
__device__ __forceinline__ float power(float l, float n) { return __builtin_amdgcn_exp2f(l * n); }
__device__ __forceinline__ float log2_decay(const float* log_decay, int head) {
    const float l = log_decay[head] * 1.4426950408889634f;
    return l < -1e30f ? -1e30f : l;
}

__device__ __forceinline__ float uniform(float v) { return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v))); }

// ---- matrix products.  An operand fragment is eight values a lane: lane l holds row (or column) l % 32 and, of a step of 16
// along the contraction, the values 8 * (l / 32) .. + 7.

template <class T> struct Frag { typedef typename Vec8<T>::type type; };

__device__ __forceinline__ floatx16 mma(half8 a, half8 b, floatx16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ floatx16 mma(Vec8<bfloat_t>::type a, Vec8<bfloat_t>::type b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ floatx16 mma(float8 a, float8 b, floatx16 c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
    return c;
}

// Accumulator row 8 * (r / 4) + 4 * (l / 32) + r % 4 sits in register r.  Where an operand's rows are handed over in the order
// perm(0), perm(1), .. (the two inner blocks of four of every sixteen exchanged), register r of the result is row
// 16 * (r / 8) + 8 * (l / 32) + r % 8: registers 0..7 and 8..15 are then each a fragment for a product along those rows.
__device__ __forceinline__ unsigned perm(unsigned i) { return (i & ~12u) | ((i & 4) << 1) | ((i & 8) >> 1); }

// ---- tiles in LDS: blocks of 32 columns, in each of which the rows lie one behind the other, in 16-byte slots that a row's
// number permutes.  Sixteen rows read at one column lie in different banks, and so do four neighbouring rows read over the
// block's width (the transposing read); a lane's addresses differ between blocks, and every 16 rows, by constants alone.
template <class T, int COLS> struct Tile {
    static constexpr int kPer = 16 / int(sizeof(T)), kSlots = COLS / kPer;   // elements a slot, slots a row
    static constexpr int kBlockSlots = 32 / kPer, kRow = kBlockSlots * 16;
    static constexpr int kBlock = (kChunk<T> + 1) * kRow;   // (a row more: the blocks of one row lie in different banks too)
    static constexpr int kBytes = COLS / 32 * kBlock;
    static __device__ __forceinline__ unsigned swizzled(unsigned row, unsigned slot) {   // of one block
        return row * kRow + (slot ^ (sizeof(T) == 2 ? (row >> 2) & 3 : (row >> 1) & 7)) * 16;
    }
    static __device__ __forceinline__ unsigned at(unsigned row, unsigned slot) { return slot / kBlockSlots * kBlock + swizzled(row, slot % kBlockSlots); }

    // Eight values of row rows + r from column 32 * block + 16 * step + 8 * half on (rows, block and step: the same in every lane;
    // rows a multiple of 32, r below 32).
    static __device__ __forceinline__ typename Frag<T>::type row8(const char* tile, int block, int step, int rows, unsigned r, unsigned half) {
        const char* p = tile + block * kBlock + rows * kRow;
        if constexpr (sizeof(T) == 2) {
            return *reinterpret_cast<const typename Frag<T>::type*>(p + swizzled(r, 2 * step + half));
        } else {
            const floatx4 lo = *reinterpret_cast<const floatx4*>(p + swizzled(r, 4 * step + 2 * half));
            const floatx4 hi = *reinterpret_cast<const floatx4*>(p + swizzled(r, 4 * step + 2 * half + 1));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
    // Column 32 * block + perm(l % 32), rows rows + 8 * (l / 32) .. + 7, for lane l (rows a multiple of 16).
    static __device__ __forceinline__ typename Frag<T>::type column8(const char* tile, int block, int rows, unsigned l) {
        const char* p = tile + block * kBlock + rows * kRow;
        if constexpr (sizeof(T) == 2) {
            // transposing read: of 16 lanes, lane j hands over four columns of row j / 4 and gets four rows of column j
            const unsigned r = 8 * (l / 32) + (l % 16) / 4;
            const unsigned b = l % 4, c = 16 * ((l / 16) % 2) + 4 * (((b & 1) << 1) | (b >> 1));
            union { short4v s[2]; typename Frag<T>::type f; } u;
            u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(p + swizzled(r, c / 8) + (c % 8) * 2));
            u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(p + swizzled(r + 4, c / 8) + (c % 8) * 2));
            return u.f;
        } else {
            const unsigned c = perm(l % 32), r = 8 * (l / 32);
            typename Frag<T>::type f;
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = *reinterpret_cast<const float*>(p + swizzled(r + i, c / 4) + (c % 4) * 4);
            return f;
        }
    }
};

// A chunk's rows of one role on their way from memory to LDS, in registers: requested while the chunk before is worked on.
// A chunk of fewer tokens lies at the tile's end: what depends on the distance to the chunk's end is then the same for all chunks.
// `column0`: the first of the tile's columns; the row has `width` (at least eight).  Rows in front of the last `valid`, and columns
// from `width` on, become zeros.  A row's last slot is read where it ends, and shifted down, so that nothing behind a row is touched.
template <class T, int COLS, int THREADS> struct Staged {
    typedef Tile<T, COLS> tile;
    static constexpr int kCount = kChunk<T> * tile::kSlots / THREADS, kStep = THREADS / tile::kSlots;
    static_assert(kCount * THREADS == kChunk<T> * tile::kSlots && kStep * tile::kSlots == THREADS, "whole rows a turn");
    uint4v r[kCount];

    static __device__ __forceinline__ int slot(unsigned tid) { return tid % tile::kSlots; }
    static __device__ __forceinline__ int row(unsigned tid, int i) { return tid / tile::kSlots + i * kStep; }

    // the chunk's row i at first + i * step bytes; |step| * rows < 2^31
    __device__ __forceinline__ void load(unsigned tid, const char* first, long long step, int valid, int column0, int width) {
        const bool down = step < 0;
        const char* low = down ? first + (valid - 1) * step : first;
        const unsigned distance = unsigned(down ? -step : step);
        const int wanted = column0 + slot(tid) * tile::kPer, last = width - tile::kPer;
        const unsigned at = unsigned(wanted < last ? wanted : last) * unsigned(sizeof(T));
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            int n = row(tid, i);
            if (valid < kChunk<T>) n = n + valid > kChunk<T> ? n + valid - kChunk<T> : 0;
            const unsigned offset = unsigned(down ? valid - 1 - n : n) * distance + at;
            __builtin_memcpy(&r[i], __builtin_assume_aligned(low + offset, sizeof(T)), 16);
        }
    }
    // in place: zeros behind the row, and what the last slot read too much of in front of its elements shifted out
    __device__ __forceinline__ void trim(unsigned tid, int valid, int column0, int width) {
        if (valid < kChunk<T>) {
#pragma unroll
            for (int i = 0; i < kCount; ++i) {
                const uint4v zero = 0u;
                r[i] = row(tid, i) + valid >= kChunk<T> ? r[i] : zero;
            }
        }
        if (width - column0 >= COLS) return;
        const int more = column0 + (slot(tid) + 1) * tile::kPer - width;   // elements of the slot that do not exist
        constexpr int kPerWord = 4 / int(sizeof(T));
        const int words = more <= 0 ? 0 : more / kPerWord, part = more <= 0 ? 0 : more % kPerWord;
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            uint4v v;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const auto word = [&](int from) {   // word `from` + words, zero behind the last
                    unsigned u = 0;
#pragma unroll
                    for (int j = from; j < 4; ++j) u = words == j - from ? r[i][j] : u;
                    return u;
                };
                v[w] = part ? word(w) >> 16 | word(w + 1) << 16 : word(w);
            }
            r[i] = v;
        }
    }
    __device__ __forceinline__ void store(unsigned tid, char* lds) const {
#pragma unroll
        for (int i = 0; i < kCount; ++i) *reinterpret_cast<uint4v*>(lds + tile::at(row(tid, i), slot(tid))) = r[i];
    }
    // whether an element is an infinity or a NaN: an exponent of ones, found by the carry out of it
    __device__ __forceinline__ bool not_finite() const {
        constexpr unsigned ones = std::is_same<T, half_t>::value ? 0x7c007c00u : std::is_same<T, bfloat_t>::value ? 0x7f807f80u : 0x7f800000u;
        constexpr unsigned low = std::is_same<T, half_t>::value ? 0x04000400u : std::is_same<T, bfloat_t>::value ? 0x00800080u : 0x00800000u;
        constexpr unsigned top = sizeof(T) == 2 ? 0x80008000u : 0x80000000u;
        unsigned found = 0;
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            const uint4v c = (r[i] & ones) + low;
            found |= c[0] | c[1] | c[2] | c[3];
        }
        return (found & top) != 0;
    }
};

template <class T> __device__ __forceinline__ typename Frag<T>::type to_frag(float8 v) { return __builtin_convertvector(v, typename Frag<T>::type); }

// w - part, eight times
template <class T> __device__ __forceinline__ float8 less(float8 w, typename Frag<T>::type part) {
    if constexpr (std::is_same<T, bfloat_t>::value) {   // (a bf16 is the upper half of a float: taken from the packed pairs as they are)
        const uint4v p = __builtin_bit_cast(uint4v, part);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            w[2 * j] -= __builtin_bit_cast(float, p[j] << 16);
            w[2 * j + 1] -= __builtin_bit_cast(float, p[j] & 0xffff0000u);
        }
        return w;
    } else {
        return w - __builtin_convertvector(part, float8);
    }
}

// The range of fp16: what becomes an operand is multiplied with a power of two that brings its largest magnitude to some 2^13, where
// that lies outside [low, 2^15].  (bf16 and fp32 have a float's range.)  Infinities and NaN do not count: they stay what they are,
// and beside them the others have to keep their range.
__device__ __forceinline__ bool in_range(float most, float low) { return most >= low && most <= 32768.f; }
__device__ __forceinline__ int exponent(float v) { return __builtin_amdgcn_frexp_expf(v); }   // v < 2^exponent, at least half of it; 0 for 0
__device__ __forceinline__ float power_of_two(float n) { return uniform(ldexpf(1.f, int(n))); }
// Of scores that are to be multiplied with values of up to 2^16: below 2^-46 they add nothing to an output.
__device__ __forceinline__ float to_range(float most) {
    const int e = 14 - exponent(most);
    return most > 0.f ? power_of_two(float(e < -126 ? -126 : e > 60 ? 60 : e)) : 1.f;
}
// Of the state, which is held under the power of two 2^now: what is to be added to `now` for a largest magnitude of 2^most (minus
// infinity: nothing there).  2^now has bounds.  Beside values of zero a state decays without end, and a power that kept up with it would
// overflow and meet those zeros; so from 2^-100 on a state fades, or where the `factor` of what is added is large by that much earlier.
// At the other end all that a float holds is brought into range.
__device__ __forceinline__ float change_of(float now, float most, float factor) {
    if (most == -__builtin_inff()) return 0.f;
    const float above = fmaxf(float(exponent(factor)), 0.f);
    return uniform(fminf(fmaxf(14.f - ceilf(most), -126.f - now), fmaxf(100.f - above, -126.f) - now));
}
__device__ __forceinline__ float finite_magnitude(float v) { return fabsf(v) < __builtin_inff() ? fabsf(v) : 0.f; }
// The largest finite magnitude in the wave's state.
template <int TILES> __device__ __forceinline__ float most_finite(const floatx16 (&x)[TILES]) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < TILES; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) m = fmaxf(m, finite_magnitude(x[i][r]));
    return lanes_max<kWave>(m);
}
__device__ __forceinline__ float most_of(half8 v) {
    half8 m = __builtin_elementwise_abs(v);
    const half4 n = __builtin_elementwise_max(__builtin_shufflevector(m, m, 0, 1, 2, 3), __builtin_shufflevector(m, m, 4, 5, 6, 7));
    return fmaxf(fmaxf(float(n[0]), float(n[1])), fmaxf(float(n[2]), float(n[3])));
}
template <int N> __device__ __forceinline__ float most8(const float8 (&v)[N]) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(v[i][j]));
    return m;
}
__device__ __forceinline__ float8 half_of(const floatx16& v, int u) {
    return u == 0 ? __builtin_shufflevector(v, v, 0, 1, 2, 3, 4, 5, 6, 7) : __builtin_shufflevector(v, v, 8, 9, 10, 11, 12, 13, 14, 15);
}

template <class T, int D, int WAVES, bool kOut>
__global__ __launch_bounds__(WAVES * 64, D <= 64 || (D == 128 && (WAVES == 4 || !kOut)) ? 2 : 1) void sweep_kernel(Sweeps a) {
    constexpr int kThreads = WAVES * 64, kTokens = kChunk<T>, kTiles = D / 32, kBlocks = kTokens / 32;
    // What is in 32 bits and becomes an operand of the outputs' products, the state that a token meets and the weighted scores, goes in
    // in two parts of the narrower types (22 bits of fp16, 16 of bf16): an output is then as far from exact arithmetic as its one
    // rounding.  In one part each it is 1.4 times as far (bf16 2.3e-3 instead of 1.66e-3, fp16 2.9e-4 instead of 2.07e-4, of the norm),
    // and the sweeps with output take 3 to 12 % less time (16 x 2048 tokens of 16 heads of 128, bf16: 175 us instead of 189).
    constexpr int kOperandParts = sizeof(T) == 2 ? 2 : 1;
    typedef Tile<T, D> tile_d;
    typedef Tile<T, WAVES * 32> tile_e;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    char* const lds_k = lds;
    char* const lds_v = lds_k + tile_d::kBytes;
    char* const lds_q = lds_v + tile_e::kBytes;      // (these two where there is output)
    char* const lds_near = lds_q + tile_d::kBytes;

    const int lane = threadIdx.x % kWave, half = lane / 32, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    long long id = blockIdx.x;
    const int which = int(id % a.count);
    id /= a.count;
    const Sweep& s = a.s[which];
    // (What the loop needs of it is read once: the compiler would otherwise load it again in every chunk, and wait.)
    const int width_d = __builtin_amdgcn_readfirstlane(s.d), width_e = __builtin_amdgcn_readfirstlane(s.e);
    const bool reverse = __builtin_amdgcn_readfirstlane(s.reverse) != 0, out_f32 = __builtin_amdgcn_readfirstlane(s.out_f32) != 0;
    const float factor_a = uniform(s.a), factor_b = uniform(s.b), factor_c = uniform(s.c);
    const int column0 = int(id % a.column_blocks) * (WAVES * 32);
    id /= a.column_blocks;
    const int head = int(id % a.heads);
    const long long slot = id / a.heads;
    if (column0 >= width_e) return;
    const long long n = sequence_of(a, slot), segment = slot - first_slot(a, n);
    const Span span = span_of(a, n);
    const bool behind = n >= (long long)a.sequences;   // tokens of no sequence: their outputs are zeros
    const long long begin = segment * (long long)a.segment;
    const long long end = begin + (long long)a.segment < span.length ? begin + (long long)a.segment : span.length;
    if (begin >= end && !(span.length == 0 && segment == 0 && !behind)) return;
    if (s.out_slots && end == span.length) return;   // (nothing starts with what the last segment adds)

    // the rows in the order of the walk: row p of the walk at first_of + p * step_of
    const auto first_of = [&](const Role& r, int size) {
        const long long first = span.first + (reverse ? span.length - 1 : 0);
        return static_cast<char*>(r.data) + ((a.cu_seqlens ? 0 : n * r.sequence) + first * r.token + (head / r.group) * r.head) * size;
    };
    const auto step_of = [&](const Role& r, int size) { return (reverse ? -r.token : r.token) * size; };
    const int e0 = wave * 32;                                            // this wave's columns of the workgroup's
    const int out_size = out_f32 ? 4 : int(sizeof(T));
    const bool whole = !out_f32 && width_e - column0 - e0 >= 32;   // 32 columns of the tensors' type to write

    if (behind) {
        if constexpr (kOut) {
            char* out = first_of(s.out, out_size);
            const int columns = width_e - column0 < WAVES * 32 ? width_e - column0 : WAVES * 32;
            for (long long p = begin + threadIdx.x / 32; p < end; p += kThreads / 32)
                for (int c = threadIdx.x % 32; c < columns; c += 32) {
                    char* at = out + p * step_of(s.out, out_size) + (column0 + c) * out_size;
                    if (out_f32) *reinterpret_cast<float*>(at) = 0.f;
                    else *reinterpret_cast<T*>(at) = T(0.f);
                }
        }
        return;
    }

    const float l2 = log2_decay(a.log_decay, head);
    floatx16 x[kTiles];
    // register r of tile i is X[32 i + 16 (r / 8) + 8 half + r % 8][column]
    const int column = column0 + e0 + perm(lane % 32);
    const auto x_row = [&](int i, int r) { return 32 * i + 16 * (r / 8) + 8 * half + r % 8; };
    const int state_size = width_d * width_e;
    {
        const float* in = s.x_in ? s.x_in + ((s.in_slots ? slot : n) * a.heads + head) * (long long)state_size : nullptr;
        const int near_column = column < width_e ? column : 0;
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
            x[i] = 0.f;
            if (in) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int d = x_row(i, r);
                    const float v = in[unsigned((d < width_d ? d : 0) * s.in_d + near_column * s.in_e)];
                    x[i][r] = d < width_d && column < width_e ? v : 0.f;
                }
            }
        }
    }

    // Decays.  The same in every lane, g^0 .. g^7, of which with a factor a lane the others are made (both at most 1, so that none
    // overflows); and in LDS, b among them, those from row to column of the scores' tiles on the diagonal, where
    // no such factor is, and which of these tiles' places count.
    float few[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) few[j] = uniform(power(l2, float(j)));
    typedef typename Frag<T>::type frag;
    typedef unsigned mask __attribute__((ext_vector_type(sizeof(frag) / 4)));
    const auto causal = [&](int u, int lane) { return lds_near + 4 * kWave * 16 + (u * kWave + lane) * int(sizeof(frag)); };
    const auto diagonal = [&](int u, int j4, int lane) { return lds_near + ((u * 2 + j4) * kWave + lane) * 16; };
    if constexpr (kOut) {
        if (wave == 0) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int j4 = 0; j4 < 2; ++j4) {
                    floatx4 v;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int apart = lane % 32 - (16 * u + 8 * half + 4 * j4 + j);
                        v[j] = apart < 0 ? 0.f : factor_b * power(l2, float(apart));
                    }
                    *reinterpret_cast<floatx4*>(diagonal(u, j4, lane)) = v;
                }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                mask m;
#pragma unroll
                for (int j = 0; j < int(sizeof(frag) / 4); ++j) {
                    const int row = 16 * u + 8 * half + j * 4 / int(sizeof(T));   // (the first of the word's)
                    const unsigned second = sizeof(T) == 2 && row + 1 <= lane % 32 ? 0xffff0000u : 0u;
                    m[j] = row > lane % 32 ? 0u : sizeof(T) == 2 ? 0x0000ffffu | second : 0xffffffffu;
                }
                *reinterpret_cast<mask*>(causal(u, lane)) = m;
            }
        }
    }
    float x_scale = 1.f;   // x holds X times this power of two (fp16 alone)

    Staged<T, D, kThreads> next_q, next_k;
    Staged<T, WAVES * 32, kThreads> next_v;
    const long long step_q = step_of(s.q, sizeof(T)), step_k = step_of(s.k, sizeof(T)), step_v = step_of(s.v, sizeof(T));
    const char* at_q = kOut ? first_of(s.q, sizeof(T)) + begin * step_q : nullptr;   // the first row of the chunk that is requested next
    const char* at_k = first_of(s.k, sizeof(T)) + begin * step_k;
    const char* at_v = first_of(s.v, sizeof(T)) + begin * step_v;
    const auto request_q = [&](unsigned tid, int valid) { next_q.load(tid, at_q, step_q, valid, 0, width_d); };
    const auto request_k = [&](unsigned tid, int valid) { next_k.load(tid, at_k, step_k, valid, 0, width_d); };
    const auto request_v = [&](unsigned tid, int valid) { next_v.load(tid, at_v, step_v, valid, column0, width_e); };
    const auto request = [&](unsigned tid, int valid) {
        request_k(tid, valid);
        request_v(tid, valid);
        if constexpr (kOut) request_q(tid, valid);
    };
    const long long step_out = kOut ? step_of(s.out, out_size) : 0;
    char* at_out = kOut ? first_of(s.out, out_size) + begin * step_out + (column0 + e0) * out_size : nullptr;
    const auto chunk_at = [&](long long p) { return int(end - p < kTokens ? end - p : kTokens); };

    // Rows of a chunk that hold an infinity or a NaN in v would spread it to the tokens before (0 * inf in a product over the
    // chunk): such a chunk is walked a token at a time.
    const bool ragged = width_d < D || width_e - column0 < WAVES * 32;
    __shared__ int bad[2];
    if (threadIdx.x == 0) bad[0] = 0;   // (the first turn's; a barrier comes before its use)
    int turn = 0;
    long long careful_until = begin;
    int valid = begin < end ? chunk_at(begin) : 0;
    if (valid > 0) request(threadIdx.x, valid);
    for (long long p = begin; p < end;) {
        // (What depends on the lane alone, addresses and powers, is formed anew for every chunk: kept over the loop it would take
        // registers that the products need.)
        unsigned tid = threadIdx.x;
        float l = l2;
        asm volatile("" : "+v"(tid), "+v"(l));
        const unsigned ulane = tid % kWave, uhalf = ulane / 32;
        const int lane = ulane, half = uhalf;
        __syncthreads();   // the chunk before has been read
        if (valid < kTokens || ragged) {
            next_k.trim(tid, valid, 0, width_d);
            next_v.trim(tid, valid, column0, width_e);
            if constexpr (kOut) next_q.trim(tid, valid, 0, width_d);
        }
        next_k.store(tid, lds_k);
        next_v.store(tid, lds_v);
        if constexpr (kOut) next_q.store(tid, lds_q);
        if (valid > 1 && __any(next_v.not_finite()) && lane == 0) bad[turn & 1] = 1;
        if (threadIdx.x == 0) bad[~turn & 1] = 0;   // (read in the turn before, used in the next)
        __syncthreads();
        if (__builtin_amdgcn_readfirstlane(bad[turn++ & 1])) {
            careful_until = p + valid;
            valid = 1;
            request(tid, 1);
            __builtin_amdgcn_s_waitcnt(0);   // (rare: no load of this branch is left to be waited for elsewhere)
            continue;
        }
        const long long after = p + valid;
        const int next_valid = after >= end ? 0 : after < careful_until ? 1 : chunk_at(after);
        at_k += valid * step_k;
        at_v += valid * step_v;
        at_q += valid * step_q;
        const int shift = kTokens - valid;   // rows of the tiles in front of the chunk's first
        frag values[kTokens / 16];   // of this wave's columns: operands of the product with the scores and of the state's update
        const auto read_values = [&] {
#pragma unroll
            for (int kk = 0; kk < kTokens / 16; ++kk) values[kk] = tile_e::column8(lds_v, wave, 16 * kk, ulane);
        };
        if constexpr (!kOut) read_values();
        // x_in of a walk from the back is the state behind the last token, and has met that token's decay already
        const float lead = reverse && p == 0 ? 0.f : 1.f;

        if constexpr (kOut) {
            if constexpr (std::is_same<T, half_t>::value) {
                float most = 0.f;
#pragma unroll
                for (int i = 0; i < kTiles; ++i) most = fmaxf(most, most8({half_of(x[i], 0), half_of(x[i], 1)}));
                if (__any(most > 32768.f) || !__any(most >= 0x1p-8f)) {
                    most = most_finite(x);
                    if (!in_range(most, 0x1p-8f)) {
                        const float now = float(exponent(x_scale) - 1);
                        const float change = fminf(change_of(now, most > 0.f ? float(exponent(most)) : -__builtin_inff(), factor_c), 126.f);
                        const float r = power_of_two(change);
                        x_scale = power_of_two(now + change);
#pragma unroll
                        for (int i = 0; i < kTiles; ++i) x[i] *= r;
                    }
                }
            }
            // along the width: the rows against the state and against the chunk's other rows
            floatx16 o[kBlocks], scores[kBlocks][kBlocks];
#pragma unroll
            for (int tb = 0; tb < kBlocks; ++tb) {
                o[tb] = 0.f;
#pragma unroll
                for (int sb = 0; sb <= tb; ++sb) scores[tb][sb] = 0.f;
            }
            // A step's operands are requested during the step before, and no earlier: left to itself the compiler requests them all
            // first and runs out of registers.
            struct Operands {
                frag k[kBlocks], q[kBlocks];
            };
            const auto operands = [&](int step) {
                Operands f;
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) {
                    f.k[b] = tile_d::row8(lds_k, step / 2, step % 2, b * 32, perm(ulane % 32), uhalf);
                    f.q[b] = tile_d::row8(lds_q, step / 2, step % 2, b * 32, ulane % 32, uhalf);
                }
                return f;
            };
            Operands now = operands(0);
#pragma unroll
            for (int step = 0; step < 2 * kTiles; ++step) {
                __builtin_amdgcn_sched_barrier(0);
                Operands then = now;
                if (step + 1 < 2 * kTiles) then = operands(step + 1);
                const float8 state = half_of(x[step / 2], step % 2);
                frag parts[kOperandParts];
                parts[0] = to_frag<T>(state);
                if constexpr (kOperandParts > 1) parts[1] = to_frag<T>(less<T>(state, parts[0]));
#pragma unroll
                for (int tb = 0; tb < kBlocks; ++tb) {
#pragma unroll
                    for (const frag& part : parts) o[tb] = mma(part, now.q[tb], o[tb]);
#pragma unroll
                    for (int sb = 0; sb <= tb; ++sb) scores[tb][sb] = mma(now.k[sb], now.q[tb], scores[tb][sb]);
                }
                now = then;
            }
            __builtin_amdgcn_sched_barrier(0);
            // (The next chunk's rows, a role at a time: all at once the requests would queue up, and the wave with them.)
            if (next_valid > 0) request_k(tid, next_valid);
            read_values();
            const int columns = width_e - column0 - e0;
#pragma unroll
            for (int tb = 0; tb < kBlocks; ++tb) {
                __builtin_amdgcn_sched_barrier(0);
                const int t = tb * 32 + lane % 32 - shift;   // (below zero: a row of zeros)
                float8 w[2 * kBlocks];
#pragma unroll
                for (int sb = 0; sb <= tb; ++sb)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        float8& to = w[2 * sb + u];
                        to = half_of(scores[tb][sb], u);
                        if (sb == tb) {
                            const floatx4 n0 = *reinterpret_cast<const floatx4*>(diagonal(u, 0, lane)), n1 = *reinterpret_cast<const floatx4*>(diagonal(u, 1, lane));
                            const float8 near = __builtin_shufflevector(n0, n1, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                            for (int j = 0; j < 8; ++j) to[j] *= near[j];
                        } else {   // g^(32 + t - s) = g^(25 + t - 16 u - 8 half) g^(7 - j)
                            to *= factor_b * power(l, float(lane % 32 + 25 - 16 * u - 8 * half));
#pragma unroll
                            for (int j = 0; j < 8; ++j) to[j] *= few[7 - j];
                        }
                    }
                float w_scale = 1.f;
                if constexpr (std::is_same<T, half_t>::value) {
                    float most = 0.f;
#pragma unroll
                    for (int j = 0; j < 2 * (tb + 1); ++j) most = fmaxf(most, most8({w[j]}));
                    if (__any(most > 32768.f) || !__any(most >= 0x1p-8f)) {
                        most = 0.f;   // (behind the diagonal there are zeros, or where a score was infinite NaN, which do not count)
#pragma unroll
                        for (int j = 0; j < 2 * (tb + 1); ++j)
#pragma unroll
                            for (int i = 0; i < 8; ++i) most = fmaxf(most, finite_magnitude(w[j][i]));
                        most = lanes_max<kWave>(most);
                        w_scale = in_range(most, 0x1p-8f) ? 1.f : to_range(most);
#pragma unroll
                        for (int j = 0; j < 2 * (tb + 1); ++j) w[j] *= w_scale;
                    }
                }
                o[tb] *= factor_a * power(l, float(t < 0 ? 0 : t) + lead) * (w_scale / x_scale);
#pragma unroll
                for (int j = 0; j < 2 * (tb + 1); ++j) {
                    asm volatile("" : "+v"(w[j]));   // (all weights first, then their parts: mixed, they need more registers than there are)
                    frag parts[kOperandParts];
                    parts[0] = to_frag<T>(w[j]);
                    if constexpr (kOperandParts > 1) parts[1] = to_frag<T>(less<T>(w[j], parts[0]));
#pragma unroll
                    for (frag weights : parts) {
                        // tokens behind the row's own: by bits, not a product with zero, for the score there may be anything
                        if (j / 2 == tb) weights = __builtin_bit_cast(frag, __builtin_bit_cast(mask, weights) & *reinterpret_cast<const mask*>(causal(j % 2, lane)));
                        o[tb] = mma(values[j], weights, o[tb]);
                    }
                }
                if (w_scale != 1.f) o[tb] *= 1.f / w_scale;
                if (tb == 0 && next_valid > 0) request_v(tid, next_valid);
                char* const row = at_out + t * step_out;
                if (t < 0) {
                } else if (whole) {
#pragma unroll
                    for (int u = 0; u < 2; ++u) store8(reinterpret_cast<T*>(row) + 16 * u + 8 * half, half_of(o[tb], u));
                } else {
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int c = 16 * u + 8 * half;
                        if (out_f32) store8(reinterpret_cast<float*>(row) + c, half_of(o[tb], u), columns - c);
                        else store8(reinterpret_cast<T*>(row) + c, half_of(o[tb], u), columns - c);
                    }
                }
            }
        }

        if (next_valid > 0) {
            if constexpr (kOut) request_q(tid, next_valid);
            else request(tid, next_valid);
        }
        float keep = power(l, float(valid - 1) + lead);
        if constexpr (std::is_same<T, half_t>::value) {
            // What the chunk adds becomes operands in two parts, the smaller of which has to keep bits that count in the state.
            float most = 0.f;
#pragma unroll
            for (int kk = 0; kk < kTokens / 16; ++kk) most = fmaxf(most, most_of(values[kk]) * power(l, float(kTokens - 16 - 16 * kk)));
            most *= fabsf(factor_c) * x_scale;
            if (__any(most > 32768.f) || !__any(most >= 0x1p-3f)) {
                most = 0.f;
#pragma unroll
                for (int kk = 0; kk < kTokens / 16; ++kk)
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        most = fmaxf(most, finite_magnitude(float(values[kk][j])) * power(l, float(kTokens - 16 - 16 * kk)));
                // in exponents: products of these magnitudes may lie outside a float's range
                most = lanes_max<kWave>(most) * __builtin_amdgcn_frexp_mantf(fabsf(factor_c));
                const float now = float(exponent(x_scale) - 1), decay = l * (float(valid - 1) + lead), of_x = most_finite(x);
                const float added = most > 0.f ? float(exponent(most) + exponent(factor_c)) + now : -__builtin_inff();
                const float larger = fmaxf(added, of_x > 0.f ? float(exponent(of_x)) + decay : -__builtin_inff());
                if (added > 15.f || larger <= -3.f) {
                    const float change = uniform(fminf(change_of(now, larger, factor_c), floorf(126.f - decay)));
                    x_scale = power_of_two(now + change);
                    keep = decay > -126.f ? ldexpf(keep, int(change)) : __builtin_amdgcn_exp2f(decay + change);   // (0 below 2^-126)
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kTiles; ++i) x[i] *= keep;
        // The state is a sum over the whole sequence, in 32 bits: of the narrower types the weighted values go into it in parts that
        // hold 22 (two of fp16) and 24 (three of bf16) bits, not in one rounding to 11 or 8.  (Two of bf16 leave the states 3e-6
        // off, relative to their norm, where sums in 32 bits alone are 2e-7 to 1e-6 off.)
        constexpr int kParts = sizeof(T) == 4 ? 1 : std::is_same<T, half_t>::value ? 2 : 3;
        struct Update {
            frag k[kTiles], v[kParts];
        };
        const auto update = [&](int kk) {
            Update f;
#pragma unroll
            for (int i = 0; i < kTiles; ++i) f.k[i] = tile_d::column8(lds_k, i, kk * 16, ulane);
            float8 w = __builtin_convertvector(values[kk], float8);
            const float to_end = factor_c * x_scale * power(l, float(kTokens - 16 * kk - 8 - 8 * half));
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] *= to_end * few[7 - j];
#pragma unroll
            for (int part = 0; part < kParts; ++part) {
                f.v[part] = to_frag<T>(w);
                if (part + 1 < kParts) w = less<T>(w, f.v[part]);
            }
            return f;
        };
        Update now = update(0);
#pragma unroll
        for (int kk = 0; kk < kTokens / 16; ++kk) {
            __builtin_amdgcn_sched_barrier(0);
            Update then = now;
            if (kk + 1 < kTokens / 16) then = update(kk + 1);
#pragma unroll
            for (int part = 0; part < kParts; ++part)
#pragma unroll
                for (int i = 0; i < kTiles; ++i) x[i] = mma(now.k[i], now.v[part], x[i]);
            now = then;
        }
        at_out += valid * step_out;
        p = after;
        valid = next_valid;
    }

    if (s.x_out && (s.out_slots || end == span.length)) {
        float* out = s.x_out + ((s.out_slots ? slot : n) * a.heads + head) * (long long)state_size;
        // (a walk from the back ends with the gradient of the state behind the first token; the initial one is a decay away)
        const float last = (reverse && !s.out_slots && span.length > 0 ? power(l2, 1.f) : 1.f) / x_scale;
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int d = x_row(i, r);
                if (d < width_d && column < width_e) out[unsigned(d * s.out_d + column * s.out_e)] = x[i][r] * last;
            }
    }
}

// From the states that each segment adds (in place, one behind the other) to the states that it starts with.  The last one's is
// not read, and not there.
struct Scan {
    Sweeps a;
    float* states;          // [slot][head][d * e]
    const float* x_in;      // [sequence][head][d * e] or null
    int size, reverse;
};

__global__ __launch_bounds__(256) void scan_kernel(Scan c) {
    const long long pair = blockIdx.y;
    const int head = int(pair % c.a.heads);
    const long long n = pair / c.a.heads;
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= c.size) return;
    const Span span = span_of(c.a, n);
    const long long slot0 = first_slot(c.a, n), segments = (span.length + c.a.segment - 1) / c.a.segment;
    const float l2 = log2_decay(c.a.log_decay, head);
    float run = c.x_in ? c.x_in[(n * c.a.heads + head) * c.size + i] : 0.f;
    const long long room = (long long)c.a.slots - slot0, some = segments > 0 ? segments : 1;   // (an empty sequence has a state too)
    const long long count = some < room ? some : room;                                           // (what cu_seqlens holds is not trusted)
    const ptrdiff_t step = ptrdiff_t(c.a.heads) * c.size;
    float* at = c.states + (slot0 * c.a.heads + head) * c.size + i;
    constexpr int kAhead = 16;   // segments whose sums are requested together
    for (long long j = 0; j < count; j += kAhead, at += kAhead * step) {
        float added[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) added[u] = j + u + 1 < count ? at[u * step] : 0.f;
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (j + u >= count) break;
            at[u * step] = run;
            run = power(l2, float(c.a.segment) - (c.reverse && j + u == 0 ? 1.f : 0.f)) * run + added[u];
        }
    }
}

// Sums the shares of the heads that have one key and value head: in [row][heads][width] floats, out one row per group.
struct Fold {
    const float* in;
    Role out;
    size_t sequences, tokens;   // rows of `in`: sequence * tokens + token
    int heads, group, width;
};

template <class T> __global__ __launch_bounds__(256) void fold_kernel(Fold f) {
    const int kv = f.heads / f.group;
    for (size_t row = blockIdx.x; row < f.sequences * f.tokens; row += gridDim.x) {
        const size_t n = row / f.tokens, t = row % f.tokens;
        for (int i = threadIdx.x; i < kv * f.width; i += 256) {
            const int h = i / f.width, c = i % f.width;
            const float* in = f.in + (row * f.heads + size_t(h) * f.group) * f.width + c;
            float v = 0.f;
            for (int g = 0; g < f.group; ++g) v += in[size_t(g) * f.width];
            static_cast<T*>(f.out.data)[ptrdiff_t(n) * f.out.sequence + ptrdiff_t(t) * f.out.token + h * f.out.head + c] = T(v);
        }
    }
}

// ---- single tokens: bound by reading and writing the state once (256 sequences of 16 heads of 128 x 128, 268 MB of state: 93 us, 5.8
// TB/s, where part of it is still in the cache behind the L2 from the token before; a copy reaches 5.1).  A workgroup has 64 columns of one state, a thread four of them of every 16th row.
struct Step {
    Role q, k, v, out;
    int heads, d, e;
    float scale;
    const float* log_decay;
    float* state;
};

template <class T> __global__ __launch_bounds__(256) void step_kernel(Step s) {
    __shared__ float qs[kMaxHead], ks[kMaxHead];
    __shared__ float sums[16][64];
    const long long n = blockIdx.x / s.heads;
    const int head = blockIdx.x % s.heads, column0 = blockIdx.y * 64;
    const auto row_of = [&](const Role& r) { return static_cast<T*>(r.data) + n * r.sequence + (head / r.group) * r.head; };
    for (int i = threadIdx.x; i < s.d; i += 256) {
        qs[i] = float(row_of(s.q)[i]) * s.scale;
        ks[i] = float(row_of(s.k)[i]);
    }
    const int x = threadIdx.x % 16, y = threadIdx.x / 16, c = column0 + 4 * x, count = s.e - c;
    const float g = power(log2_decay(s.log_decay, head), 1.f);
    float v[4], o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = j < count ? float(row_of(s.v)[c + j]) : 0.f;
    __syncthreads();
    float* state = s.state + (n * s.heads + head) * s.d * (long long)s.e + c;
    if (count >= 4) {
#pragma unroll 4
        for (int d = y; d < s.d; d += 16) {
            floatx4 r;
            __builtin_memcpy(&r, __builtin_assume_aligned(state + (long long)d * s.e, 4), 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                r[j] = g * r[j] + ks[d] * v[j];
                o[j] += qs[d] * r[j];
            }
            __builtin_memcpy(__builtin_assume_aligned(state + (long long)d * s.e, 4), &r, 16);
        }
    } else if (count > 0) {
        for (int d = y; d < s.d; d += 16) {
#pragma unroll
            for (int j = 0; j < 3; ++j)
                if (j < count) {
                    const float r = g * state[(long long)d * s.e + j] + ks[d] * v[j];
                    o[j] += qs[d] * r;
                    state[(long long)d * s.e + j] = r;
                }
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) sums[y][4 * x + j] = o[j];
    __syncthreads();
    if (threadIdx.x < 64 && column0 + int(threadIdx.x) < s.e) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) t += sums[i][threadIdx.x];
        row_of(s.out)[column0 + threadIdx.x] = T(t);
    }
}

// ---- host side

constexpr size_t kMaxThreads = 0xffffffffu;   // along one axis of a launch
constexpr size_t kWhole = size_t(1) << 41;   // a segment that holds any sequence

int padded(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

bool valid_shape(const flstm_decay_attention* p) {
    return p && valid_dtype(p->dtype) && p->heads > 0 && p->kv_heads > 0 && p->heads % p->kv_heads == 0 && p->heads <= 65535 && p->dk >= kMinHead &&
           p->dv >= kMinHead && p->dk <= kMaxHead && p->dv <= kMaxHead && p->scale == p->scale && p->log_decay &&
           p->sequences < (size_t(1) << 31) && p->tokens < (size_t(1) << 40) && (!p->cu_seqlens || p->tokens < (size_t(1) << 31));
}

// Tokens a workgroup walks.  A walk over a whole sequence reads everything once, but few heads leave most of the chip idle; cut
// into segments it reads keys and values twice, for what each segment adds to the state comes first.  Measured with heads of 128
// x 128, bf16 (us, whole walks / segments): forward, 192 workgroups of 2048 tokens 160 / 188, 128 of them 149 / 151, four of 4096
// 275 / 54, four heads of eight packed sequences of 2530 tokens on average (8192 the longest) 540 / 92; packed, 192 workgroups with up to
// 4096 tokens 276 / 227, since the longest decides; gradients (three walks), 128 workgroups of 2048 tokens 266 / 257, the four of 4096
// 276 / 65, the packed eight 545 / 161.
// Segments are as long as leaves 512 workgroups, which is two a CU and one round (256 where a workgroup's registers fill a CU):
// 131072 tokens of 8 heads, fp16, take 492 us in segments of 2048, 512 of 1024, 528 of 4096.  Of packed sequences, whose last segments are
// not full, three quarters of one more each are reckoned with: 12 of them with 16 heads take 227 us so, 265 in
// segments of 1408.
// Eight chunks are walked as a whole: three launches take as long.  512 tokens, bf16, whole walks / segments: 4 heads 41 / 42, 16 heads 42 /
// 49, four sequences of 16 heads 43 / 58, gradients 39 / 44, 40 / 54, 43 / 82; of 1024 tokens 73 / 44, 74 / 51, 75 / 71 and 73 / 48, 73 /
// 62, 78 / 130.  256 tokens of fp32, where a chunk has 32, are as many chunks (300 of 16 heads 86 / 62, gradients 86 / 63).
// Segments shorter than 256 tokens come with fewer workgroups than 512: more of them are states to be written, scanned and read for few
// tokens, and backward there are three walks.  Segments of 64 tokens / of 256, fp32, forward and gradients together: seven packed
// sequences of up to 200 tokens, 6 heads of 40 x 65, 121 / 199; one of 512, 16 heads of 128 x 128, 147 / 256.  (Four of 512 with 16 heads,
// bf16, gradients: 133 / 81.)
size_t segment_of(const flstm_decay_attention* p, bool backward) {
    const size_t blocks = size_t(p->heads) * ceil_div(size_t(p->dv), 128), walks = p->sequences * blocks;
    const size_t chunk = p->dtype == FLSTM_OP_F32 ? kChunk<float> : kChunk<half_t>;
    if (walks == 0 || p->tokens <= 8 * chunk || walks >= (backward ? 128 : p->cu_seqlens ? 256 : 129)) return kWhole;
    const size_t room = p->dk > 128 || p->dv > 128 ? 256 : 512;
    size_t segment;
    if (p->cu_seqlens) {
        const size_t partial = walks * 3 / 4;
        segment = ceil_div(p->tokens * blocks, partial * 2 < room ? room - partial : room / 2);
    } else {
        segment = ceil_div(p->tokens, walks < room ? room / walks : 1);
    }
    if (segment < 256) {
        const size_t least = ceil_div(p->cu_seqlens ? p->tokens * blocks : p->tokens * walks, room / (backward ? 3 : 2));
        segment = segment > least ? segment : least < 256 ? least : 256;
    }
    return round_up(segment, 64);
}
size_t slots_of(const flstm_decay_attention* p, bool backward) {
    const size_t segment = segment_of(p, backward);
    if (p->cu_seqlens) return p->tokens / segment + p->sequences + 1;
    return p->sequences * (p->tokens ? ceil_div(p->tokens, segment) : 1);
}
size_t states_bytes(const flstm_decay_attention* p, bool backward) {
    const size_t slots = slots_of(p, backward);
    const bool split = p->tokens > segment_of(p, backward);
    return split ? round_up(slots * p->heads * size_t(p->dk) * p->dv * sizeof(float), 256) : 0;
}
// Whether a chunk's rows lie within 32-bit offsets.
bool reachable(const flstm_decay_attention* p, const flstm_rows& r) {
    return p->tokens <= 1 || (r.token < (ptrdiff_t(1) << 23) && r.token > -(ptrdiff_t(1) << 23));
}

size_t rows_of(const flstm_decay_attention* p) { return p->cu_seqlens ? p->tokens : p->sequences * p->tokens; }
size_t shares_bytes(const flstm_decay_attention* p, int width) {
    return p->heads == p->kv_heads ? 0 : round_up(rows_of(p) * p->heads * size_t(width) * sizeof(float), 256);
}

flstm_rows or_none(const flstm_rows* r) { return r ? *r : flstm_rows{}; }
Role role(const flstm_rows& r, int group) { return Role{r.data, r.sequence, r.token, r.head, group}; }

Sweeps sweeps_of(const flstm_decay_attention* p, bool backward) {
    Sweeps a{};
    a.sequences = p->sequences; a.tokens = p->tokens; a.slots = slots_of(p, backward); a.segment = segment_of(p, backward);
    a.cu_seqlens = p->cu_seqlens; a.heads = p->heads; a.log_decay = p->log_decay;
    return a;
}

template <class T, int D, int WAVES, bool kOut> int launch_sweeps(Sweeps a, hipStream_t stream) {
    int widest = 0;
    for (int i = 0; i < a.count; ++i) widest = a.s[i].e > widest ? a.s[i].e : widest;
    a.column_blocks = int(ceil_div(size_t(widest), WAVES * 32));
    const size_t grid = a.slots * size_t(a.heads) * a.column_blocks * a.count;
    if (grid == 0) return 0;
    if (grid > kMaxThreads / (WAVES * 64)) return FLSTM_E_TOO_LARGE;
    constexpr int lds = Tile<T, D>::kBytes * (kOut ? 2 : 1) + Tile<T, WAVES * 32>::kBytes + (kOut ? kWave * (4 * 16 + 2 * 8 * int(sizeof(T))) : 0);
    const auto kernel = sweep_kernel<T, D, WAVES, kOut>;
    if (lds > 65536) {
        const hipError_t rc = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (rc != hipSuccess) return int(rc);
    }
    kernel<<<unsigned(grid), WAVES * 64, lds, stream>>>(a);
    return launched();
}

// Waves a workgroup, of 32 columns each.  (Two of 256 rows would have to hold more than their registers.)
int waves_of(int d, int e) { return e <= 64 && d <= 128 ? 2 : 4; }

// Runs the sweeps of `a`, those of one padded width in one launch.
int run_sweeps(const Sweeps& all, flstm_op_dtype dtype, bool out, hipStream_t stream) {
    for (const int d : {64, 128, 256})
        for (const int waves : {2, 4}) {
            Sweeps a = all;
            a.count = 0;
            for (int i = 0; i < all.count; ++i)
                if (padded(all.s[i].d) == d && waves_of(d, all.s[i].e) == waves) a.s[a.count++] = all.s[i];
            if (a.count == 0) continue;
            const int rc = with_type(dtype, [&](auto zero) {
                typedef decltype(zero) T;
                const auto go = [&](auto width) {
                    constexpr int D = decltype(width)::value;
                    if (out) return waves == 2 ? launch_sweeps<T, D, 2, true>(a, stream) : launch_sweeps<T, D, 4, true>(a, stream);
                    return waves == 2 ? launch_sweeps<T, D, 2, false>(a, stream) : launch_sweeps<T, D, 4, false>(a, stream);
                };
                if (d == 256) {
                    if (out) return launch_sweeps<T, 256, 4, true>(a, stream);
                    return launch_sweeps<T, 256, 4, false>(a, stream);
                }
                if (d == 64) return go(std::integral_constant<int, 64>());
                return go(std::integral_constant<int, 128>());
            });
            if (rc != 0) return rc;
        }
    return 0;
}

int run_scan(const Sweeps& a, float* states, const float* x_in, int size, int reverse, hipStream_t stream) {
    if (a.sequences * a.heads > 65535) return FLSTM_E_TOO_LARGE;
    if (a.sequences == 0) return 0;
    const Scan c{a, states, x_in, size, reverse};
    scan_kernel<<<dim3(unsigned(ceil_div(size_t(size), 256)), unsigned(a.sequences * a.heads)), 256, 0, stream>>>(c);
    return launched();
}

}  // namespace
}  // namespace flstm_hip

using namespace flstm_hip;

extern "C" size_t flstm_decay_attention_workspace_bytes(const flstm_decay_attention* p, int backward) {
    if (!valid_shape(p)) return 0;
    return backward ? 2 * states_bytes(p, true) + shares_bytes(p, p->dk) + shares_bytes(p, p->dv) : states_bytes(p, false);
}

extern "C" int flstm_decay_attention_forward(const flstm_decay_attention* p, const flstm_rows* q_, const flstm_rows* k_, const flstm_rows* v_,
                                             const float* state_in, const flstm_rows* o_, float* state_out, void* workspace, void* stream) {
    if (!valid_shape(p)) return FLSTM_E_INVALID;
    const flstm_rows q = or_none(q_), k = or_none(k_), v = or_none(v_), o = or_none(o_);
    if (rows_of(p) > 0 && (!q.data || !k.data || !v.data || !o.data)) return FLSTM_E_INVALID;
    if (states_bytes(p, false) > 0 && !workspace) return FLSTM_E_INVALID;
    if (!reachable(p, q) || !reachable(p, k) || !reachable(p, v)) return FLSTM_E_TOO_LARGE;
    if (p->sequences == 0 && !p->cu_seqlens) return 0;
    hipStream_t stream_ = static_cast<hipStream_t>(stream);
    const int group = p->heads / p->kv_heads;
    Sweeps a = sweeps_of(p, false);
    Sweep& s = a.s[0];
    a.count = 1;
    s = Sweep{role(q, 1), role(k, group), role(v, group), role(o, 1), p->dk, p->dv, 0, 0, state_in, state_out, p->dv, 1, p->dv, 1, 0, 0,
              p->scale, p->scale, 1.f};
    if (states_bytes(p, false) > 0) {
        float* states = static_cast<float*>(workspace);
        s.x_in = nullptr; s.x_out = states; s.out_slots = 1;
        int rc = run_sweeps(a, p->dtype, false, stream_);
        if (rc == 0) rc = run_scan(a, states, state_in, p->dk * p->dv, 0, stream_);
        if (rc != 0) return rc;
        s.x_in = states; s.in_slots = 1; s.x_out = state_out; s.out_slots = 0;
    }
    return run_sweeps(a, p->dtype, true, stream_);
}

extern "C" int flstm_decay_attention_backward(const flstm_decay_attention* p, const flstm_rows* d_o_, const flstm_rows* q_, const flstm_rows* k_, const flstm_rows* v_,
                                              const float* state_in, const float* d_state_out, const flstm_rows* dq_, const flstm_rows* dk_,
                                              const flstm_rows* dv_, float* d_state_in, void* workspace, void* stream) {
    if (!valid_shape(p)) return FLSTM_E_INVALID;
    const flstm_rows d_o = or_none(d_o_), q = or_none(q_), k = or_none(k_), v = or_none(v_), dq = or_none(dq_), dk = or_none(dk_), dv = or_none(dv_);
    if (rows_of(p) > 0 && (!d_o.data || !q.data || !k.data || !v.data)) return FLSTM_E_INVALID;
    if (flstm_decay_attention_workspace_bytes(p, 1) > 0 && !workspace) return FLSTM_E_INVALID;
    if (!reachable(p, d_o) || !reachable(p, q) || !reachable(p, k) || !reachable(p, v)) return FLSTM_E_TOO_LARGE;
    if (p->sequences == 0 && !p->cu_seqlens) return 0;
    hipStream_t stream_ = static_cast<hipStream_t>(stream);
    const int group = p->heads / p->kv_heads;
    char* room = static_cast<char*>(workspace);
    const bool split = states_bytes(p, true) > 0;
    float* const states = reinterpret_cast<float*>(room);                      // S at the segments' starts
    float* const adjoints = reinterpret_cast<float*>(room + states_bytes(p, true));  // A behind the segments' ends
    char* const shares_k = room + 2 * states_bytes(p, true);
    char* const shares_v = shares_k + shares_bytes(p, p->dk);
    const Role rq = role(q, 1), rk = role(k, group), rv = role(v, group), rdo = role(d_o, 1);
    const auto shared = [&](const flstm_rows& r, char* room, int width) {   // where a sweep leaves a head's share
        if (group == 1 || !r.data) return role(r, 1);
        return Role{room, ptrdiff_t(p->tokens) * p->heads * width, ptrdiff_t(p->heads) * width, width, 1};
    };
    const int f32 = group > 1;
    const Sweep to_q{rdo, rv, rk, role(dq, 1), p->dv, p->dk, 0, 0, state_in, nullptr, 1, p->dv, 1, p->dv, 0, 0, p->scale, p->scale, 1.f};
    const Sweep to_v{rk, rq, rdo, shared(dv, shares_v, p->dv), p->dk, p->dv, f32, 1, d_state_out, d_state_in, p->dv, 1, p->dv, 1, 0, 0,
                     1.f, p->scale, p->scale};
    const Sweep to_k{rv, rdo, rq, shared(dk, shares_k, p->dk), p->dv, p->dk, f32, 1, d_state_out, nullptr, 1, p->dv, 1, p->dv, 0, 0,
                     1.f, p->scale, p->scale};
    Sweeps a = sweeps_of(p, true);
    a.count = 0;
    if (split) {
        // what each segment adds to S and to A, then what each starts with
        Sweep s = to_v;   // (k, q, do) from the back: A
        s.x_in = nullptr; s.x_out = adjoints; s.out_slots = 1;
        a.s[a.count++] = s;
        if (dq.data) {
            s = Sweep{rq, rk, rv, Role{}, p->dk, p->dv, 0, 0, nullptr, states, p->dv, 1, p->dv, 1, 0, 1, 1.f, 1.f, 1.f};
            a.s[a.count++] = s;
        }
        int rc = run_sweeps(a, p->dtype, false, stream_);
        if (rc == 0) rc = run_scan(a, adjoints, d_state_out, p->dk * p->dv, 1, stream_);
        if (rc == 0 && dq.data) rc = run_scan(a, states, state_in, p->dk * p->dv, 0, stream_);
        if (rc != 0) return rc;
    }
    const auto add = [&](Sweep s, const float* at) {
        if (split) { s.x_in = at; s.in_slots = 1; }
        a.s[a.count++] = s;
    };
    a.count = 0;
    if (dq.data) add(to_q, states);
    if (dv.data) add(to_v, adjoints);
    if (dk.data) add(to_k, adjoints);
    int rc = run_sweeps(a, p->dtype, true, stream_);
    if (rc == 0 && !dv.data && d_state_in) {   // nothing but the state is asked of this walk
        a.count = 0;
        add(to_v, adjoints);
        rc = run_sweeps(a, p->dtype, false, stream_);
    }
    if (rc != 0 || group == 1 || rows_of(p) == 0) return rc;
    const auto fold = [&](const flstm_rows& r, char* shares, int width) {
        if (!r.data) return 0;
        const size_t rows = rows_of(p), tokens = p->cu_seqlens ? rows : p->tokens;
        const Fold f{reinterpret_cast<const float*>(shares), role(r, 1), rows / tokens, tokens, p->heads, group, width};
        return with_type(p->dtype, [&](auto zero) {
            fold_kernel<decltype(zero)><<<unsigned(rows < (1u << 20) ? rows : (1u << 20)), 256, 0, stream_>>>(f);
            return launched();
        });
    };
    rc = fold(dk, shares_k, p->dk);
    return rc != 0 ? rc : fold(dv, shares_v, p->dv);
}

extern "C" int flstm_decay_attention_step(const flstm_decay_attention* p, const flstm_rows* q_, const flstm_rows* k_, const flstm_rows* v_, const flstm_rows* o_,
                                          float* state, void* stream) {
    if (!valid_shape(p)) return FLSTM_E_INVALID;
    if (p->sequences == 0) return 0;
    const flstm_rows q = or_none(q_), k = or_none(k_), v = or_none(v_), o = or_none(o_);
    if (!q.data || !k.data || !v.data || !o.data || !state) return FLSTM_E_INVALID;
    const size_t grid = p->sequences * size_t(p->heads);
    if (grid > kMaxThreads / 256) return FLSTM_E_TOO_LARGE;
    const int group = p->heads / p->kv_heads;
    const Step s{role(q, 1), role(k, group), role(v, group), role(o, 1), p->heads, p->dk, p->dv, p->scale, p->log_decay, state};
    return with_type(p->dtype, [&](auto zero) {
        step_kernel<decltype(zero)><<<dim3(unsigned(grid), unsigned(ceil_div(size_t(p->dv), 64))), 256, 0, static_cast<hipStream_t>(stream)>>>(s);
        return launched();
    });
}
