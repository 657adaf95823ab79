// A gated linear recurrence over the tokens of sequences (lm_ops.h): prompts, gradients, single tokens.
//
//   c_t = f_t c_{t-1} + (1 - f_t) x_t,  f = sigmoid(forget),  y_t = c_t or sigmoid(gate_t) c_t
// Channels do not meet, so that a lane walks channels of its own along the tokens, and all of it is bound by memory.  Where sequences and
// channels are too few to fill the chip (the rule is at `split`), sequences are cut into segments of a few tokens a wave, held in registers: what a segment
// makes of a state, a factor and a sum, is published, those in front of it are read, and the segment goes on from the state that they
// give.  Every tensor is so read and written once, and the order of all sums depends on sizes alone.
// Of f and 1 - f the smaller one is computed and the other's part left whole, c = x + f (c - x) or c = c + (1 - f)(x - c): a
// rounding of 1 - small would be the same at every token of a channel that mostly keeps its state, and add up over its memory.  Nor is it a product of factors
// near one that segments publish, for the same reason, but what that lacks to one.
// The backward pass needs the states in front of all tokens.  They are walked again from the states that the forward pass leaves
// every kBatch tokens, in 32 bits: y, rounded to 16 bits, would not give forget's gradient, which is a difference of states.
// With a gate: 256 sequences of 1024 tokens and channels, fp16, walked whole, 420 us forward (5.3 TB/s) and 732 backward (5.2); one of 131072 tokens,
// bf16, in segments, 237 forward (4.8 TB/s, where the vector units' five functions a token and channel are as much of a bound).
#include <type_traits>

#include "lm_device.h"

namespace flstm_hip {
namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 16;   // tokens between two saved states, and on their way to a lane at a time
constexpr int kGroup = 8;    // segments whose work is put together, and such groups once more

struct Rows {
    void* data;
    ptrdiff_t sequence, token;   // elements
};

struct Recurrence {
    size_t sequences, tokens, segment;   // segment: tokens
    unsigned slots, each;                // segments' slots in all, and of a sequence that is not packed
    const int* cu_seqlens;
    unsigned width;
    Rows x, forget, gate, y;      // gate.data: null without an output gate
    Rows dy, dx, dforget, dgate;
    const float *initial, *d_final;   // (sequences, width) or null
    float *final, *d_initial;
    float* saved;             // [batch slot][width]
    unsigned* ticket;         // workgroups that have begun; behind it, whether one has waited in vain
    u64* made[3];             // [slot][width]: what segments, groups of kGroup segments and groups of these make of a state
};

// Sequence n's tokens, whatever cu_seqlens holds; n == sequences: those behind the last.
struct Span { long long first, length; };
__device__ __forceinline__ Span span_of(const Recurrence& a, long long n) {
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
// Pieces of `size` tokens of a sequence have consecutive slots.  Packed: from first / size + n on, which leaves each enough of them
// without a sum over the sequences before.
__device__ __forceinline__ long long first_slot(const Recurrence& a, long long n, long long size) {
    if (!a.cu_seqlens) return n * (a.tokens ? ((long long)a.tokens + size - 1) / size : 1);
    return span_of(a, n).first / size + n;
}
__device__ __forceinline__ long long sequence_of(const Recurrence& a, long long slot) {
    if (!a.cu_seqlens) return unsigned(slot) / a.each;
    // the last n whose first slot is not behind this one: all lanes look at as many places at a time
    long long lo = 0, hi = (long long)a.sequences;
    while (lo < hi) {
        const long long step = (hi - lo + kWave - 1) / kWave, n = lo + (long long)(threadIdx.x % kWave + 1) * step;
        const int many = __popcll(__ballot(n <= hi && first_slot(a, n, (long long)a.segment) <= slot));
        lo += many * step;
        hi = lo + step - 1 < hi ? lo + step - 1 : hi;
    }
    return lo;
}

// A sigmoid as its smaller side s, in (0, 1/2], and which one that is.  fp32 tensors: the exponential's argument in two parts and a
// quotient corrected once, which the hardware's functions alone would leave some units of 2^-24 off.
template <class T> __device__ __forceinline__ float small_sigmoid(float u) {
    const float v = -fabsf(u);
    float e;
    if constexpr (sizeof(T) == 4) {
        constexpr float kLog2e = 1.4426950408889634f, kRest = 1.925963033500576e-08f;
        const float t = v * kLog2e, rest = __builtin_fmaf(v, kLog2e, -t) + v * kRest;
        const bool tiny = t < -100.f;   // (the hardware's exponential has no numbers below 2^-126)
        e = __builtin_amdgcn_exp2f(tiny ? t + 64.f : t) * (tiny ? 0x1p-64f : 1.f);
        if (t > -1000.f) e = __builtin_fmaf(e, rest * 0.6931471805599453f, e);
        const float d = 1.f + e, r = __builtin_amdgcn_rcpf(d), q = e * r;
        return __builtin_fmaf(__builtin_fmaf(-q, d, e), r, q);
    }
    e = __builtin_amdgcn_exp2f(v * 1.4426950408889634f);
    return e * __builtin_amdgcn_rcpf(1.f + e);
}
struct Factor {
    float small;   // the smaller of f and 1 - f
    bool keeps;    // 1 - f is
};
template <class T> __device__ __forceinline__ Factor factor_of(float forget) { return Factor{small_sigmoid<T>(forget), forget > 0.f}; }
__device__ __forceinline__ float keep(Factor f) { return f.keeps ? 1.f - f.small : f.small; }     // f
__device__ __forceinline__ float kept(Factor f, float v) { return f.keeps ? __builtin_fmaf(-f.small, v, v) : f.small * v; }   // f v
__device__ __forceinline__ float lost(Factor f, float v) { return f.keeps ? f.small * v : __builtin_fmaf(-f.small, v, v); }   // (1 - f) v
__device__ __forceinline__ float stepped(Factor f, float c, float x) {
    const float base = f.keeps ? c : x, other = f.keeps ? x : c;
    return __builtin_fmaf(f.small, other - base, base);
}
__device__ __forceinline__ float small(Factor f) { return f.small; }
// The same as one word, the smaller one as -f or 1 - f, and in an operation or two less, with the same results.  (Where a factor is computed again from its gate
// the form above takes fewer registers: this one spills in the forward pass of 16-bit tensors.)
struct Held {
    float way;
    __device__ __forceinline__ bool keeps() const { return __builtin_bit_cast(int, way) >= 0; }
};
__device__ __forceinline__ Factor factor(Factor f) { return f; }
__device__ __forceinline__ Factor factor(Held f) { return Factor{fabsf(f.way), f.keeps()}; }
__device__ __forceinline__ Held held(Held f) { return f; }
__device__ __forceinline__ Held held(Factor f) { return Held{__builtin_copysignf(f.small, f.keeps ? 1.f : -1.f)}; }
__device__ __forceinline__ float kept(Held f, float v) { return __builtin_fmaf(-f.way, v, f.keeps() ? v : 0.f); }
__device__ __forceinline__ float lost(Held f, float v) { return __builtin_fmaf(f.way, v, f.keeps() ? 0.f : v); }
__device__ __forceinline__ float stepped(Held f, float c, float x) { return __builtin_fmaf(f.way, x - c, f.keeps() ? c : x); }
__device__ __forceinline__ float small(Held f) { return fabsf(f.way); }
template <class T> __device__ __forceinline__ float sigmoid(float u) {
    if constexpr (sizeof(T) == 2) return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(u * -1.4426950408889634f));
    const float s = small_sigmoid<T>(u);
    return u > 0.f ? 1.f - s : s;
}

// What is the same for all lanes, in scalar registers; kScalar: and so a row's address, which takes 64-bit addresses of all rows on their way out of the vector
// registers.  (The long walk has room for them, and is a tenth slower without: 425 us instead of 473 for 256 x 1024 x 1024 fp16.)
__device__ __forceinline__ long long scalar(long long v) {
    const unsigned lo = __builtin_amdgcn_readfirstlane(unsigned(v)), hi = __builtin_amdgcn_readfirstlane(unsigned(v >> 32));
    return (long long)(u64(hi) << 32 | lo);
}
template <bool kScalar> __device__ __forceinline__ const char* address(const char* row, unsigned at) {
    if constexpr (kScalar) asm("" : "+s"(row));
    return row + at;
}

// A workgroup's piece of a sequence: one segment (or, n == sequences, the tokens behind the last, which get zeros).
struct Piece {
    long long n, begin, end, first;   // tokens of the sequence; the sequence's first token in a packed tensor
    long long slot;
    bool last;
};
__device__ __forceinline__ bool piece_of(const Recurrence& a, long long slot, Piece& p) {
    p.slot = slot = scalar(slot);
    p.n = scalar(sequence_of(a, slot));
    const Span span = span_of(a, p.n);
    const long long index = slot - first_slot(a, p.n, (long long)a.segment);
    p.begin = scalar(index * (long long)a.segment);
    const long long length = scalar(span.length);
    if (index < 0 || (index > 0 && p.begin >= length)) return false;
    p.end = length - p.begin < (long long)a.segment ? length : p.begin + (long long)a.segment;
    p.first = scalar(span.first);
    p.last = p.end == length;
    return true;
}
// Where a piece's tensor begins at `token` of its sequence.  The same for all lanes: a lane's channels are a 32-bit offset to it, in bytes, so that the
// addresses of a walk are the scalar unit's.
template <class T> __device__ __forceinline__ char* row_of(const Recurrence& a, const Rows& r, const Piece& p, long long token) {
    return static_cast<char*>(r.data) + (a.cu_seqlens ? (p.first + token) * r.token : p.n * r.sequence + token * r.token) * ptrdiff_t(sizeof(T));
}

// C neighbouring channels at a time; the last lane of an odd width has one channel in common with its neighbour, and both
// compute and write the same.
template <int BYTES> struct Word;
template <> struct Word<2> { typedef unsigned short type; };
template <> struct Word<4> { typedef unsigned type; };
template <> struct Word<8> { typedef u64 type; };
template <class T, int C> struct Few {
    typename Word<C * sizeof(T)>::type word;   // as they lie in memory: 16-bit ones in pairs
    __device__ __forceinline__ float operator[](int j) const {
        typedef T V __attribute__((ext_vector_type(C)));
        return float(__builtin_bit_cast(V, word)[j]);
    }
    // What was made of the word so far is not kept: it is converted again, where it is used again.
    __device__ __forceinline__ void forget() { asm volatile("" : "+v"(word)); }
};
template <class T, int C, bool kScalar> __device__ __forceinline__ Few<T, C> load_few(const char* row, unsigned at) {
    Few<T, C> v;
    __builtin_memcpy(&v.word, __builtin_assume_aligned(address<kScalar>(row, at), sizeof(T)), sizeof(v.word));
    return v;
}
// kPassing: past the caches, for tensors that they do not hold.
template <class T, int C, bool kScalar, bool kPassing> __device__ __forceinline__ void store_few(char* row, unsigned at, const float* v) {
    typedef typename Word<C * sizeof(T)>::type __attribute__((aligned(sizeof(T)))) Unaligned;
    T r[C];
#pragma unroll
    for (int j = 0; j < C; ++j) r[j] = T(v[j]);
    typename Word<C * sizeof(T)>::type word;
    __builtin_memcpy(&word, r, sizeof(word));
    Unaligned* to = reinterpret_cast<Unaligned*>(const_cast<char*>(address<kScalar>(row, at)));
    if constexpr (kPassing) __builtin_nontemporal_store(word, to);
    else *to = word;
}
// A row of states.
template <int C> __device__ __forceinline__ Few<float, C> load_state(const float* states, long long row, const Recurrence& a, unsigned c) {
    return load_few<float, C, true>(reinterpret_cast<const char*>(states + row * a.width), c * 4);
}
template <int C> __device__ __forceinline__ void store_state(float* states, long long row, const Recurrence& a, unsigned c, const float* v) {
    store_few<float, C, true, false>(reinterpret_cast<char*>(states + row * a.width), c * 4, v);
}
// kBatch tokens of a tensor; those that do not exist are zeros.
template <class T, int C, bool kScalar, bool kFull>
__device__ __forceinline__ void load_batch(Few<T, C> (&v)[kBatch], const Recurrence& a, const Rows& r, const Piece& p, long long t, unsigned at, int count) {
    const char* row = row_of<T>(a, r, p, t);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
        if (kFull || i < count) v[i] = load_few<T, C, kScalar>(row + i * r.token * ptrdiff_t(sizeof(T)), at);
        else v[i].word = 0;
    }
}

// A lane's channels, `block` lanes of a workgroup beside one another.  (Lanes behind the last do its work again.)
template <int C> __device__ __forceinline__ unsigned channel_of(const Recurrence& a, unsigned block, unsigned lanes, unsigned lane) {
    const unsigned c = (block * lanes + lane) * C;
    return c + C > a.width ? a.width - C : c;
}

// A segment's first channel; the last of an odd width is not alone.
template <int C> __device__ __forceinline__ unsigned first_channel(const Recurrence& a, unsigned block) {
    const unsigned c = block * kWave * C;
    return c + C > a.width ? a.width - C : c;
}

// A token's gradients, each where it is wanted, from the states in front of it and behind it; s: f_{t+1} G_{t+1}, then f_t G_t.
struct Gradients {
    char *dx, *dforget, *dgate;   // rows, or null
};
template <class T, int C, bool kGate, bool kScalar, bool kPassing, class F, class U>
__device__ __forceinline__ void gradients(const Recurrence& a, const Gradients& to, int i, unsigned at, F&& factor, const U& u, const Few<T, C>& x, const Few<T, C>& d,
                                          const Few<T, C>& g, const float (&before)[C], const float (&after)[C], float (&s)[C]) {
    float of_x[C], of_forget[C], of_gate[C];
#pragma unroll
    for (int j = 0; j < C; ++j) {
        const auto k = factor(u[j]);
        float dc = d[j];
        if constexpr (kGate) {
            const Factor o = factor_of<T>(g[j]);
            of_gate[j] = dc * after[j] * (o.small * (1.f - o.small));
            dc *= keep(o);
        }
        const float total = dc + s[j];
        of_x[j] = lost(k, total);
        of_forget[j] = total * (before[j] - x[j]) * (small(k) * (1.f - small(k)));
        s[j] = kept(k, total);
    }
    constexpr ptrdiff_t kSize = sizeof(T);
    if (to.dx) store_few<T, C, kScalar, kPassing>(to.dx + i * a.dx.token * kSize, at, of_x);
    if (to.dforget) store_few<T, C, kScalar, kPassing>(to.dforget + i * a.dforget.token * kSize, at, of_forget);
    if constexpr (kGate)
        if (to.dgate) store_few<T, C, kScalar, kPassing>(to.dgate + i * a.dgate.token * kSize, at, of_gate);
}
template <class T> __device__ __forceinline__ Gradients gradients_at(const Recurrence& a, const Piece& p, long long t) {
    const auto row = [&](const Rows& r) { return r.data ? row_of<T>(a, r, p, t) : nullptr; };
    return Gradients{row(a.dx), row(a.dforget), row(a.dgate)};
}
// Zeros for the tokens behind the last sequence, every `step`th of them.
template <class T, int C> __device__ __forceinline__ void clear_rows(const Recurrence& a, const Rows& r, const Piece& p, unsigned at, int first, int step) {
    const float zeros[C] = {};
    if (r.data)
        for (long long t = p.begin + first; t < p.end; t += step) store_few<T, C, false, false>(row_of<T>(a, r, p, t), at, zeros);
}

// ---- whole sequences: a lane walks from the first token to the last.  A workgroup has neighbouring channels of one sequence, up to kWalkLanes lanes, so
// that rows are read as wholes.  (Measured with rows' addresses in scalar registers, forward: 473 us, workgroups of 64 lanes 487, lanes of four channels, half
// as many waves, 513.)

constexpr unsigned kWalkLanes = 256;

template <class T, int C, bool kGate, bool kPassing> __global__ __launch_bounds__(kWalkLanes) void forward_kernel(Recurrence a, unsigned blocks) {
    Piece p;
    if (!piece_of(a, blockIdx.x / blocks, p)) return;
    const unsigned c = channel_of<C>(a, blockIdx.x % blocks, blockDim.x, threadIdx.x), at = c * unsigned(sizeof(T));
    if (p.n == (long long)a.sequences) return clear_rows<T, C>(a, a.y, p, at, 0, 1);
    float s[C];
#pragma unroll
    for (int j = 0; j < C; ++j) s[j] = a.initial ? a.initial[p.n * a.width + c + j] : 0.f;
    long long saved = first_slot(a, p.n, kBatch);
    const auto batch = [&](long long t, auto full, int count) {
        constexpr bool kFull = decltype(full)::value;
        Few<T, C> u[kBatch], x[kBatch], g[kBatch];
        load_batch<T, C, false, kFull>(u, a, a.forget, p, t, at, count);
        load_batch<T, C, false, kFull>(x, a, a.x, p, t, at, count);
        if constexpr (kGate) load_batch<T, C, false, kFull>(g, a, a.gate, p, t, at, count);
        if (a.saved) store_state<C>(a.saved, saved++, a, c, s);
        char* y = row_of<T>(a, a.y, p, t);
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (!kFull && i >= count) continue;
            float o[C];
#pragma unroll
            for (int j = 0; j < C; ++j) {
                s[j] = stepped(factor_of<T>(u[i][j]), s[j], x[i][j]);
                o[j] = s[j];
                if constexpr (kGate) o[j] *= sigmoid<T>(g[i][j]);
            }
            store_few<T, C, false, kPassing>(y + i * a.y.token * ptrdiff_t(sizeof(T)), at, o);
        }
    };
    long long t = 0;
    for (; t + kBatch <= p.end; t += kBatch) batch(t, std::true_type(), kBatch);
    if (t < p.end) batch(t, std::false_type(), int(p.end - t));
    if (a.final) store_state<C>(a.final, p.n, a, c, s);
}

// From the last token to the first, G_t = sigmoid(gate_t) dy_t + f_{t+1} G_{t+1}: kBatch tokens' states again, then their gradients.
template <class T, int C, bool kGate, bool kPassing> __global__ __launch_bounds__(kWalkLanes) void backward_kernel(Recurrence a, unsigned blocks) {
    Piece p;
    if (!piece_of(a, blockIdx.x / blocks, p)) return;
    const unsigned c = channel_of<C>(a, blockIdx.x % blocks, blockDim.x, threadIdx.x), at = c * unsigned(sizeof(T));
    if (p.n == (long long)a.sequences) {
        clear_rows<T, C>(a, a.dx, p, at, 0, 1);
        clear_rows<T, C>(a, a.dforget, p, at, 0, 1);
        return clear_rows<T, C>(a, a.dgate, p, at, 0, 1);
    }
    float s[C];
#pragma unroll
    for (int j = 0; j < C; ++j) s[j] = a.d_final ? a.d_final[p.n * a.width + c + j] : 0.f;
    const long long saved = first_slot(a, p.n, kBatch);
    const auto batch = [&](long long t, auto full, int count) {
        constexpr bool kFull = decltype(full)::value;
        Few<T, C> u[kBatch], x[kBatch], d[kBatch], g[kBatch];
        load_batch<T, C, false, kFull>(u, a, a.forget, p, t, at, count);
        load_batch<T, C, false, kFull>(x, a, a.x, p, t, at, count);
        load_batch<T, C, false, kFull>(d, a, a.dy, p, t, at, count);
        if constexpr (kGate) load_batch<T, C, false, kFull>(g, a, a.gate, p, t, at, count);
        const Few<float, C> before = load_state<C>(a.saved, saved + t / kBatch, a, c);
        float state[kBatch + 1][C];
#pragma unroll
        for (int j = 0; j < C; ++j) state[0][j] = before[j];
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
#pragma unroll
            for (int j = 0; j < C; ++j) state[i + 1][j] = stepped(factor_of<T>(u[i][j]), state[i][j], x[i][j]);
        const Gradients to = gradients_at<T>(a, p, t);
#pragma unroll
        for (int i = kBatch - 1; i >= 0; --i)
            if (kFull || i < count) gradients<T, C, kGate, false, kPassing>(a, to, i, at, factor_of<T>, u[i], x[i], d[i], g[i], state[i], state[i + 1], s);
    };
    const long long whole = p.end / kBatch * kBatch;
    if (whole < p.end) batch(whole, std::false_type(), int(p.end - whole));
    for (long long t = whole - kBatch; t >= 0; t -= kBatch) batch(t, std::true_type(), kBatch);
    if (a.d_initial) store_state<C>(a.d_initial, p.n, a, c, s);
}

// ---- segments
//
// A workgroup has one segment, kBatch tokens a wave, of kWave * C channels.  Workgroups take their segments in order, so that those whose work one
// waits for have begun before it, and each publishes before it waits: every wait ends.  What a segment needs of those in front
// of it is what the groups of groups, the groups in the last of these, and the segments in the last group make of a state; the last segment
// of a group publishes the group's, as soon as it has its own group's.  A published pair is one word, which is its own flag: words are kNothing before.
// (With cu_seqlens that do not ascend a group may have no last segment.  What is not there after a second reads as NaN, and nobody waits from then on.)

constexpr u64 kNothing = ~u64(0);
constexpr unsigned kMostPolls = 1u << 20;

struct Made {
    float factor, sum;   // state -> factor * state + sum
};
__device__ __forceinline__ float of(const Made& m, float state) { return __builtin_fmaf(m.factor, state, m.sum); }
// The same as it is handed on: 1 - factor, or of a factor up to 1/2 its negative.  A product of factors near one, each rounded to a multiple of 2^-24, is off by as
// many of these as it has factors, all in one direction where the tokens' gates are alike; so what it lacks to one is added up beside it, from the tokens on.  (The
// states of 41000 tokens of fp32 with forget gates of 8 to 12 are off by at most 12 times 2^-24; with products alone by 28 to 4600.)
struct Packed {
    float way, sum;
};
__device__ __forceinline__ Made unpacked(const Packed& p) { return Made{(Held{p.way}.keeps() ? 1.f : 0.f) - p.way, p.sum}; }
// What tokens, or pieces of them, make of a state, one behind the other.
struct Walk {
    float factor = 1.f, sum = 0.f, less = 0.f;   // less: 1 - factor, as long as that is less than 1/2
    template <class F> __device__ __forceinline__ void leaves(F f) {
        less = __builtin_fmaf(small(f), factor, less);   // (where 1 - f is not the smaller one, factor is 1/2 at most from here on)
        factor = kept(f, factor);
    }
    __device__ __forceinline__ void behind(const Packed& p) {
        const Made next = unpacked(p);
        less = __builtin_fmaf(fabsf(p.way), factor, less);
        factor *= next.factor;
        sum = of(next, sum);
    }
    __device__ __forceinline__ Packed packed() const { return Packed{factor > 0.5f ? less : -factor, sum}; }
};
// A row of published pairs: the same for all lanes, a lane's word `at` bytes behind it.
__device__ __forceinline__ u64* word_of(const u64* row, unsigned at) {
    return reinterpret_cast<u64*>(const_cast<char*>(address<true>(reinterpret_cast<const char*>(row), at)));
}
__device__ __forceinline__ void publish(u64* row, unsigned at, Packed p) {
    if (p.way != p.way) p.way = __builtin_nanf("");   // (not kNothing's)
    __hip_atomic_store(word_of(row, at), __builtin_bit_cast(u64, p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ u64 look(const u64* row, unsigned at) { return __hip_atomic_load(word_of(row, at), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// What the pairs of `count` rows from `row` on, `step` words apart, make of a state, one after the other.
__device__ __forceinline__ Walk read_made(const u64* row, ptrdiff_t step, long long count, unsigned at, unsigned* in_vain) {
    Walk m;
    constexpr int kAhead = kGroup - 1;   // all there are of segments and groups (one more: registers that cost fp32 tensors with a gate a workgroup a CU, 6 % of the time)
    for (long long i = 0; i < count; i += kAhead, row += kAhead * step) {
        u64 v[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (i + k < count) v[k] = look(row + k * step, at);
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (i + k < count) {
                for (unsigned poll = 1; v[k] == kNothing && poll <= kMostPolls; ++poll) {
                    __builtin_amdgcn_s_sleep(1);
                    v[k] = look(row + k * step, at);
                    if (poll % 256 == 0 && __hip_atomic_load(in_vain, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) break;
                    if (poll == kMostPolls) __hip_atomic_store(in_vain, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
                m.behind(__builtin_bit_cast(Packed, v[k]));
            }
    }
    return m;
}

// Between the two passes over a segment's tokens its forget gates stay in their words: 16-bit ones as they came, since their factors again cost less than
// the registers of 32-bit ones (a third workgroup on a CU), fp32 ones as the smaller of f and 1 - f, negative where that is f.
template <class T, int C> __device__ __forceinline__ void hold_factors(Few<T, C>& u) {
    if constexpr (sizeof(T) == 4) {
        float s[C];
#pragma unroll
        for (int j = 0; j < C; ++j) s[j] = held(factor_of<T>(u[j])).way;
        __builtin_memcpy(&u.word, s, sizeof(s));
    }
}
template <class T> __device__ __forceinline__ auto held_factor(float u) {
    if constexpr (sizeof(T) == 4) return Held{u};
    else return factor_of<T>(u);
}
// A token that is none, which keeps the state.
template <class T, int C> __device__ __forceinline__ Few<T, C> no_token() {
    T v[C];
#pragma unroll
    for (int j = 0; j < C; ++j) v[j] = T(__builtin_inff());
    Few<T, C> r;
    __builtin_memcpy(&r.word, v, sizeof(v));
    return r;
}

// Which segment a workgroup has, from the first (the last, where kBack) on; false: none.
template <bool kBack> __device__ __forceinline__ bool take_piece(const Recurrence& a, unsigned blocks, Piece& p, unsigned& block) {
    __shared__ unsigned ticket;
    if (threadIdx.x == 0) ticket = atomicAdd(a.ticket, 1u);
    __syncthreads();
    const unsigned mine = __builtin_amdgcn_readfirstlane(ticket), slot = mine / blocks;
    block = mine - slot * blocks;
    return piece_of(a, kBack ? a.slots - 1 - slot : slot, p);
}

// The state in front of the wave's tokens (behind them, where kBack), from what its tokens make of one and all in front of them; `from` is the
// sequence's first.  Publishes the segment's.  A wave and its neighbour see to half of the channels each, one a lane.
template <int C, int W, bool kBack> __device__ __forceinline__ void state_at(const Recurrence& a, const Piece& p, unsigned c0, unsigned c, const Walk (&own)[C],
                                                                             const float* from, float (&s)[C]) {
    constexpr int kChannels = kWave * C, kRoles = W / 2;
    constexpr long long kSize = W * kBatch;
    __shared__ Packed parts[W][kChannels], before[kRoles + 1][kChannels];
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), order = kBack ? W - 1 - wave : wave;
#pragma unroll
    for (int j = 0; j < C; ++j) parts[order][c - c0 + j] = own[j].packed();
    const long long place = p.begin / kSize;                                                 // in the sequence
    const long long at = kBack ? (span_of(a, p.n).length - 1) / kSize - place : place;       // as the walk goes
    const long long few = at % kGroup, group = at / kGroup, few_groups = group % kGroup, groups = group / kGroup;
    const int role = wave / 2, ch = wave % 2 * kWave + lane;
    const bool mine = ch < kChannels && c0 + ch < a.width;
    const unsigned word = (c0 + ch) * unsigned(sizeof(u64));
    const ptrdiff_t width = a.width;
    const auto row_at = [&](int level, long long slot) { return a.made[level] + scalar(slot * width); };
    __syncthreads();
    Packed all{};
    if (role == 0 && mine) {
        Walk here;
#pragma unroll
        for (int w = 0; w < W; ++w) here.behind(parts[w][ch]);
        all = here.packed();
        publish(row_at(0, p.slot), word, all);
        Walk walk = read_made(row_at(0, kBack ? p.slot + few : p.slot - few), kBack ? -width : width, few, word, a.ticket + 1);
        before[0][ch] = walk.packed();
        walk.behind(all);
        all = walk.packed();
        if (few == kGroup - 1) publish(row_at(1, first_slot(a, p.n, kSize * kGroup) + group), word, all);
    } else if (mine) {
        if (role == 1) before[1][ch] = read_made(row_at(1, first_slot(a, p.n, kSize * kGroup) + group - few_groups), width, few_groups, word, a.ticket + 1).packed();
        if (role > 1 || kRoles == 2) {   // the groups of groups, in as many parts as there are roles for
            constexpr int kParts = kRoles == 2 ? 1 : kRoles - 2;
            const int part = kRoles == 2 ? 0 : role - 2;
            const long long some = (groups + kParts - 1) / kParts, begin = part * some, left = groups - begin < some ? groups - begin : some;
            before[2 + part][ch] = read_made(row_at(2, first_slot(a, p.n, kSize * kGroup * kGroup) + begin), width, left, word, a.ticket + 1).packed();
        }
    }
    __syncthreads();
    if (role == 0 && mine && few == kGroup - 1 && few_groups == kGroup - 1) {
        Walk walk;
        walk.behind(before[1][ch]);
        walk.behind(all);
        publish(row_at(2, first_slot(a, p.n, kSize * kGroup * kGroup) + groups), word, walk.packed());
    }
#pragma unroll
    for (int j = 0; j < C; ++j) {
        s[j] = from ? from[p.n * a.width + c + j] : 0.f;
#pragma unroll
        for (int r = 2; r < (kRoles == 2 ? 3 : kRoles); ++r) s[j] = of(unpacked(before[r][c - c0 + j]), s[j]);
        s[j] = of(unpacked(before[0][c - c0 + j]), of(unpacked(before[1][c - c0 + j]), s[j]));
        for (int w = 0; w < order; ++w) s[j] = of(unpacked(parts[w][c - c0 + j]), s[j]);
    }
}

template <class T, int C, bool kGate, bool kPassing, int W>
__global__ __launch_bounds__(W * kWave, C == 2 && sizeof(T) == 2 ? 6 : 3) void split_forward_kernel(Recurrence a, unsigned blocks) {
    Piece p;
    unsigned block;
    if (!take_piece<false>(a, blocks, p, block)) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const unsigned c0 = first_channel<C>(a, block), lane = threadIdx.x % kWave;
    const unsigned c = c0 + (lane + 1) * C > a.width ? a.width - C : c0 + lane * C, at = c * unsigned(sizeof(T));
    if (p.n == (long long)a.sequences) return clear_rows<T, C>(a, a.y, p, at, wave, W);
    const long long t = p.begin + wave * kBatch;
    const int count = p.end - t < 0 ? 0 : p.end - t < kBatch ? int(p.end - t) : kBatch;
    Few<T, C> u[kBatch], x[kBatch], g[kBatch];
    const auto load = [&](auto full) {
        constexpr bool kFull = decltype(full)::value;
        load_batch<T, C, true, kFull>(u, a, a.forget, p, t, at, count);
        load_batch<T, C, true, kFull>(x, a, a.x, p, t, at, count);
        if constexpr (kGate) load_batch<T, C, true, kFull>(g, a, a.gate, p, t, at, count);
        if constexpr (!kFull)
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
                if (i >= count) u[i] = no_token<T, C>();
    };
    if (count == kBatch) load(std::true_type());
    else load(std::false_type());
    // Of half of the tokens the factors stay in LDS, which is three workgroups' for that: two functions less a token (257 us instead of 277 for 131072 tokens
    // of 1024 channels with a gate, bf16, where the vector units are the bound).
    constexpr int kInLds = sizeof(T) == 2 ? kBatch / 2 : 0;
    __shared__ Few<float, C> factors[kInLds ? kInLds : 1][kInLds ? W * kWave : 1];
    Walk made[C];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
        hold_factors<T, C>(u[i]);
        float way[C];
#pragma unroll
        for (int j = 0; j < C; ++j) {
            const Factor k = factor(held_factor<T>(u[i][j]));   // (as Held, 20 registers more of fp32 tensors without a gate, and 4 % of the time)
            way[j] = held(k).way;
            made[j].leaves(k);
            made[j].sum = stepped(k, made[j].sum, x[i][j]);
        }
        if (i < kInLds) __builtin_memcpy(&factors[i][threadIdx.x].word, way, sizeof(way));
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
        u[i].forget();
        x[i].forget();
    }
    float s[C];
    state_at<C, W, false>(a, p, c0, c, made, a.initial, s);
    if (a.saved && count > 0) store_state<C>(a.saved, first_slot(a, p.n, kBatch) + t / kBatch, a, c, s);
    char* y = row_of<T>(a, a.y, p, t);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
        if (i >= count) continue;
        float o[C];
        Few<float, C> in_lds{};
        if (i < kInLds) in_lds = factors[i][threadIdx.x];
#pragma unroll
        for (int j = 0; j < C; ++j) {
            s[j] = i < kInLds ? stepped(Held{in_lds[j]}, s[j], x[i][j]) : stepped(held_factor<T>(u[i][j]), s[j], x[i][j]);
            o[j] = s[j];
            if constexpr (kGate) o[j] *= sigmoid<T>(g[i][j]);
        }
        store_few<T, C, true, kPassing>(y + i * a.y.token * ptrdiff_t(sizeof(T)), at, o);
    }
    if (p.last && a.final && wave == W - 1) store_state<C>(a.final, p.n, a, c, s);   // (waves behind the end keep the state)
}

template <class T, int C, bool kGate, bool kPassing, int W> __global__ __launch_bounds__(W * kWave) void split_backward_kernel(Recurrence a, unsigned blocks) {
    Piece p;
    unsigned block;
    if (!take_piece<true>(a, blocks, p, block)) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const unsigned c0 = first_channel<C>(a, block), lane = threadIdx.x % kWave;
    const unsigned c = c0 + (lane + 1) * C > a.width ? a.width - C : c0 + lane * C, at = c * unsigned(sizeof(T));
    if (p.n == (long long)a.sequences) {
        clear_rows<T, C>(a, a.dx, p, at, wave, W);
        clear_rows<T, C>(a, a.dforget, p, at, wave, W);
        return clear_rows<T, C>(a, a.dgate, p, at, wave, W);
    }
    const long long t = p.begin + wave * kBatch;
    const int count = p.end - t < 0 ? 0 : p.end - t < kBatch ? int(p.end - t) : kBatch;
    Few<T, C> u[kBatch], x[kBatch], g[kBatch], d[kBatch];
    const auto load = [&](auto full) {
        constexpr bool kFull = decltype(full)::value;
        load_batch<T, C, true, kFull>(u, a, a.forget, p, t, at, count);
        load_batch<T, C, true, kFull>(d, a, a.dy, p, t, at, count);
        if constexpr (kGate) load_batch<T, C, true, kFull>(g, a, a.gate, p, t, at, count);
        load_batch<T, C, true, kFull>(x, a, a.x, p, t, at, count);
        if constexpr (!kFull)
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
                if (i >= count) u[i] = no_token<T, C>();
    };
    if (count == kBatch) load(std::true_type());
    else load(std::false_type());
    Few<float, C> first{};
    if (count > 0) first = load_state<C>(a.saved, first_slot(a, p.n, kBatch) + t / kBatch, a, c);
    constexpr int kInLds = sizeof(T) == 2 ? kBatch : 0;   // tokens whose factors stay in LDS
    __shared__ Few<float, C> factors[kInLds ? kInLds : 1][kInLds ? W * kWave : 1];
    Walk made[C];
#pragma unroll
    for (int i = kBatch - 1; i >= 0; --i) {
        hold_factors<T, C>(u[i]);
        float way[C];
#pragma unroll
        for (int j = 0; j < C; ++j) {
            const auto k = held_factor<T>(u[i][j]);
            way[j] = held(k).way;
            float dc = d[i][j];
            if constexpr (kGate) dc *= sigmoid<T>(g[i][j]);
            made[j].leaves(k);
            made[j].sum = kept(k, made[j].sum + dc);
        }
        if (i < kInLds) __builtin_memcpy(&factors[i][threadIdx.x].word, way, sizeof(way));
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
        u[i].forget();
        d[i].forget();
        if constexpr (kGate) g[i].forget();
    }
    float s[C];
    state_at<C, W, true>(a, p, c0, c, made, a.d_final, s);
    float state[kBatch + 1][C];
#pragma unroll
    for (int j = 0; j < C; ++j) state[0][j] = first[j];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
        x[i].forget();   // (the states from here on)
#pragma unroll
        for (int j = 0; j < C; ++j) {
            if constexpr (kInLds > 0) state[i + 1][j] = stepped(Held{factors[i][threadIdx.x][j]}, state[i][j], x[i][j]);
            else state[i + 1][j] = stepped(held_factor<T>(u[i][j]), state[i][j], x[i][j]);
        }
    }
    const Gradients to = gradients_at<T>(a, p, t);
#pragma unroll
    for (int i = kBatch - 1; i >= 0; --i)
        if (i < count) {
            if constexpr (kInLds > 0) gradients<T, C, kGate, true, kPassing>(a, to, i, at, held_factor<float>, factors[i][threadIdx.x], x[i], d[i], g[i], state[i], state[i + 1], s);
            else gradients<T, C, kGate, true, kPassing>(a, to, i, at, held_factor<T>, u[i], x[i], d[i], g[i], state[i], state[i + 1], s);
        }
    if (p.begin == 0 && wave == 0 && a.d_initial) store_state<C>(a.d_initial, p.n, a, c, s);
}

// Nothing published, no workgroup begun.
__global__ __launch_bounds__(kThreads) void clear_kernel(u64* words, size_t count) {
    for (size_t i = size_t(blockIdx.x) * kThreads + threadIdx.x; i < count; i += size_t(gridDim.x) * kThreads) words[i] = i == 0 ? 0 : kNothing;
}

// One token of every sequence: vectors of eight channels.
template <class T, bool kGate> __global__ __launch_bounds__(kThreads) void step_kernel(Recurrence a, unsigned vectors, size_t first) {
    const unsigned item = blockIdx.x * kThreads + threadIdx.x, in_launch = item / vectors;
    const size_t n = first + in_launch, c = size_t(item - in_launch * vectors) * 8;
    if (n >= a.sequences) return;
    const int many = a.width - c < 8 ? int(a.width - c) : 8;
    const auto row = [&](const Rows& r) { return static_cast<T*>(r.data) + (long long)n * r.sequence + c; };
    float* state = a.final + n * a.width + c;
    const float8 x = load8(row(a.x), many), u = load8(row(a.forget), many);
    float8 s = load8(state, many), g = 0.f;
    if constexpr (kGate) g = load8(row(a.gate), many);
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = stepped(factor_of<T>(u[j]), s[j], x[j]);
    store8(state, s, many);
    if constexpr (kGate)
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] *= sigmoid<T>(g[j]);
    store8(row(a.y), s, many);
}

// ---- host side

constexpr size_t kWhole = size_t(1) << 40;   // a segment that holds any sequence
constexpr size_t kMostThreads = 0xffffffffu;

bool valid_shape(const flstm_recurrence* p) {
    return p && valid_dtype(p->dtype) && p->sequences < (size_t(1) << 31) && p->width < (size_t(1) << 28) &&
           p->tokens < (p->cu_seqlens ? size_t(1) << 31 : size_t(1) << 39);
}
// Whether sequences are cut into segments.  Walked whole, a sequence takes some 2.3 us for every 16 tokens forward and 5 backward, until its lanes fill the
// chip; cut, some 18 and 24 us to begin with, of which the clearing of the published words is a launch.  Measured (us, cut / whole, forward and backward, fp16 with
// a gate, 1024 channels): one sequence of 64 tokens 18 / 15 and 25 / 25, of 128 18 / 22 and 24 / 44, of 512 19 / 75 and 25 / 158; 64 of 128 27 / 25 and 43 /
// 48, of 2048 237 / 417 and 427 / 724; 128 of 128 43 / 32 and 63 / 56, of 1024 233 / 234 and 416 / 402; 256 of 512 224 / 214 and 400 / 380.
// Of packed sequences the longest decides how long the whole walk takes, and is not known: 200 of up to 2000 tokens 387 / 543 and 688 / 934, 400 of up
// to 1000 429 / 474 and 758 / 823, but 200 of up to 100 51 / 34 and 67 / 55.  All of these are of lengths spread evenly up to the longest: the rule knows the mean alone,
// and one long sequence among many short ones is walked whole however long it is (199 of 50 tokens and one of 10000: 1511 and 3103 us; 511 of 10 and one of
// 60000: 10720 and 19393).
bool split(const flstm_recurrence* p) {
    const size_t lanes = round_up(ceil_div(p->width, 2), kWave);
    if (p->tokens <= 64) return false;
    if (p->sequences * lanes < 65536) return true;
    return p->cu_seqlens && p->sequences * lanes < 262144 && p->tokens >= 128 * p->sequences;
}
size_t rows_of(const flstm_recurrence* p) { return p->cu_seqlens ? p->tokens : p->sequences * p->tokens; }
size_t slots_of(const flstm_recurrence* p, size_t size) {
    if (p->cu_seqlens) return p->tokens / size + p->sequences + 1;
    return p->sequences * (p->tokens ? ceil_div(p->tokens, size) : 1);
}
// Waves of a segment's workgroup.  A lane holds a segment's tokens in registers, more of them backwards.
constexpr int kForwardWaves = 8, kBackwardWaves = 4;
size_t segment_of(const flstm_recurrence* p, bool backward) { return split(p) ? (backward ? kBackwardWaves : kForwardWaves) * kBatch : kWhole; }
// Words of the workspace: the workgroups' counter (and nothing, to 16 bytes), then what segments and groups make of a state.
size_t words_of(const flstm_recurrence* p, bool backward) {
    if (!split(p)) return 0;
    size_t words = 2;
    for (size_t i = 0, size = segment_of(p, backward); i < 3; ++i, size *= kGroup) words += slots_of(p, size) * p->width;
    return words;
}
Rows rows(const flstm_rows* r) { return r ? Rows{r->data, r->sequence, r->token} : Rows{}; }

Recurrence recurrence_of(const flstm_recurrence* p, const flstm_rows* x, const flstm_rows* forget, const flstm_rows* gate, bool backward) {
    Recurrence a{};
    a.sequences = p->sequences; a.tokens = p->tokens; a.segment = segment_of(p, backward);
    a.each = unsigned(p->tokens ? ceil_div(p->tokens, a.segment) : 1);
    a.cu_seqlens = p->cu_seqlens; a.width = unsigned(p->width);
    a.x = rows(x); a.forget = rows(forget); a.gate = rows(gate);
    return a;
}

constexpr size_t kMostKept = size_t(32) << 20;   // bytes of a tensor that the caches hold

template <class T, int C, bool kGate, bool kPassing, bool kBack> int launch(const flstm_recurrence* p, Recurrence a, void* workspace, hipStream_t stream) {
    constexpr int W = kBack ? kBackwardWaves : kForwardWaves;
    const size_t words = words_of(p, kBack), pairs = ceil_div(p->width, size_t(C)), slots = slots_of(p, a.segment);
    const size_t lanes = words ? kWave : pairs < kWalkLanes ? round_up(pairs, kWave) : kWalkLanes, blocks = ceil_div(pairs, lanes);
    if (slots > kMostThreads / (words ? W * kWave : lanes) / blocks) return FLSTM_E_TOO_LARGE;
    const unsigned grid = unsigned(slots * blocks);
    a.slots = unsigned(slots);
    if (words) {
        u64* at = static_cast<u64*>(workspace);
        a.ticket = reinterpret_cast<unsigned*>(at);
        at += 2;
        for (size_t i = 0, size = a.segment; i < 3; at += slots_of(p, size) * p->width, ++i, size *= kGroup) a.made[i] = at;
        const size_t clears = ceil_div(words, kThreads * 4);
        clear_kernel<<<unsigned(clears < 2048 ? clears : 2048), kThreads, 0, stream>>>(static_cast<u64*>(workspace), words);
        if (const int rc = launched()) return rc;
        if constexpr (kBack) split_backward_kernel<T, C, kGate, kPassing, W><<<grid, W * kWave, 0, stream>>>(a, unsigned(blocks));
        else split_forward_kernel<T, C, kGate, kPassing, W><<<grid, W * kWave, 0, stream>>>(a, unsigned(blocks));
    } else {
        if constexpr (kBack) backward_kernel<T, C, kGate, kPassing><<<grid, unsigned(lanes), 0, stream>>>(a, unsigned(blocks));
        else forward_kernel<T, C, kGate, kPassing><<<grid, unsigned(lanes), 0, stream>>>(a, unsigned(blocks));
    }
    return launched();
}
template <bool kBack> int run(const flstm_recurrence* p, const Recurrence& a, void* workspace, hipStream_t stream) {
    return with_type(p->dtype, [&](auto zero) {
        typedef decltype(zero) T;
        const bool passing = rows_of(p) * p->width * sizeof(T) > kMostKept;
        if (p->width == 1) return a.gate.data ? launch<T, 1, true, false, kBack>(p, a, workspace, stream) : launch<T, 1, false, false, kBack>(p, a, workspace, stream);
        if (a.gate.data) return passing ? launch<T, 2, true, true, kBack>(p, a, workspace, stream) : launch<T, 2, true, false, kBack>(p, a, workspace, stream);
        return passing ? launch<T, 2, false, true, kBack>(p, a, workspace, stream) : launch<T, 2, false, false, kBack>(p, a, workspace, stream);
    });
}

}  // namespace
}  // namespace flstm_hip

using namespace flstm_hip;

extern "C" size_t flstm_gated_recurrence_workspace_bytes(const flstm_recurrence* p, int backward) {
    return valid_shape(p) ? words_of(p, backward != 0) * sizeof(u64) : 0;
}
extern "C" size_t flstm_gated_recurrence_saved_rows(const flstm_recurrence* p) { return valid_shape(p) ? slots_of(p, kBatch) : 0; }

extern "C" int flstm_gated_recurrence_forward(const flstm_recurrence* p, const flstm_rows* x, const flstm_rows* forget, const flstm_rows* gate,
                                              const float* state_in, const flstm_rows* y, float* state_out, float* saved, void* workspace,
                                              void* stream) {
    if (!valid_shape(p)) return FLSTM_E_INVALID;
    if (p->width == 0 || (p->sequences == 0 && !p->cu_seqlens)) return 0;
    Recurrence a = recurrence_of(p, x, forget, gate, false);
    a.y = rows(y); a.initial = state_in; a.final = state_out; a.saved = saved;
    if (rows_of(p) > 0 && (!a.x.data || !a.forget.data || !a.y.data)) return FLSTM_E_INVALID;
    if (words_of(p, false) > 0 && !workspace) return FLSTM_E_INVALID;
    return run<false>(p, a, workspace, static_cast<hipStream_t>(stream));
}

extern "C" int flstm_gated_recurrence_backward(const flstm_recurrence* p, const flstm_rows* dy, const flstm_rows* x, const flstm_rows* forget,
                                               const flstm_rows* gate, const float* saved, const float* d_state_out, const flstm_rows* dx,
                                               const flstm_rows* dforget, const flstm_rows* dgate, float* d_state_in, void* workspace, void* stream) {
    if (!valid_shape(p)) return FLSTM_E_INVALID;
    if (p->width == 0 || (p->sequences == 0 && !p->cu_seqlens)) return 0;
    Recurrence a = recurrence_of(p, x, forget, gate, true);
    a.dy = rows(dy); a.dx = rows(dx); a.dforget = rows(dforget); a.dgate = rows(dgate);
    a.saved = const_cast<float*>(saved); a.d_final = d_state_out; a.d_initial = d_state_in;
    if (rows_of(p) > 0 && (!a.x.data || !a.forget.data || !a.dy.data || !saved)) return FLSTM_E_INVALID;
    if ((a.dgate.data && !a.gate.data) || (words_of(p, true) > 0 && !workspace)) return FLSTM_E_INVALID;
    return run<true>(p, a, workspace, static_cast<hipStream_t>(stream));
}

extern "C" int flstm_gated_recurrence_step(const flstm_recurrence* p, const flstm_rows* x, const flstm_rows* forget, const flstm_rows* gate,
                                           const flstm_rows* y, float* state, void* stream) {
    if (!valid_shape(p)) return FLSTM_E_INVALID;
    if (p->width == 0 || p->sequences == 0) return 0;
    Recurrence a{};
    a.sequences = p->sequences; a.width = unsigned(p->width); a.final = state;
    a.x = rows(x); a.forget = rows(forget); a.gate = rows(gate); a.y = rows(y);
    if (!a.x.data || !a.forget.data || !a.y.data || !state) return FLSTM_E_INVALID;
    const size_t vectors = ceil_div(p->width, 8), most = (size_t(1) << 31) / vectors;   // sequences a launch
    return with_type(p->dtype, [&](auto zero) {
        typedef decltype(zero) T;
        hipStream_t s = static_cast<hipStream_t>(stream);
        for (size_t first = 0; first < p->sequences; first += most) {
            const size_t some = p->sequences - first < most ? p->sequences - first : most;
            a.sequences = first + some;
            const unsigned grid = unsigned(ceil_div(some * vectors, kThreads));
            if (a.gate.data) step_kernel<T, true><<<grid, kThreads, 0, s>>>(a, unsigned(vectors), first);
            else step_kernel<T, false><<<grid, kThreads, 0, s>>>(a, unsigned(vectors), first);
            if (const int rc = launched()) return rc;
        }
        return 0;
    });
}
