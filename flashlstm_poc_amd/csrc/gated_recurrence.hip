// A gated linear recurrence over the tokens of sequences (lm_ops.h): prompts, gradients, single tokens.
//
//   c_t = f_t c_{t-1} + (1 - f_t) x_t,  f = sigmoid(forget),  y_t = c_t or sigmoid(gate_t) c_t
// Channels do not meet, so that a lane walks channels of its own along the tokens, and all of it is bound by memory.  Where sequences and
// channels are too few for the chip, sequences are cut into segments: what each makes of a state (a factor and what is added),
// those joined in order, and the walk itself from the right states.
// Of f and 1 - f the smaller one is computed and the other's part left whole, c = x + f (c - x) or c = c + (1 - f)(x - c): a
// rounding of 1 - small would be the same at every token of a channel that mostly keeps its state, and add up over its memory.
// The backward pass needs the states in front of all tokens.  They are walked again from the states that the forward pass leaves
// every kBatch tokens, in 32 bits: y, rounded to 16 bits, would not give forget's gradient, which is a difference of states.
#include <type_traits>

#include "lm_device.h"

namespace flstm_hip {
namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 16;   // tokens between two saved states, and on their way to a lane at a time

struct Rows {
    void* data;
    ptrdiff_t sequence, token;   // elements
};

struct Recurrence {
    size_t sequences, tokens, segment, segments;   // segment: tokens, a multiple of kBatch; segments: slots in all
    const int* cu_seqlens;
    unsigned width;
    Rows x, forget, gate, y;      // gate.data: null without an output gate
    Rows dy, dx, dforget, dgate;
    const float *initial, *d_final;   // (sequences, width) or null
    float *final, *d_initial;
    float* saved;             // [batch slot][width]
    float2* carried;          // [segment slot][width]: factor and sum, then the state in front of (behind) the segment in .x
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
    if (!a.cu_seqlens) return slot / (a.tokens ? ((long long)a.tokens + (long long)a.segment - 1) / (long long)a.segment : 1);
    long long lo = 0, hi = (long long)a.sequences;   // the last n whose first slot is not behind this one
    while (lo < hi) {
        const long long mid = (lo + hi + 1) / 2;
        if (first_slot(a, mid, (long long)a.segment) <= slot) lo = mid; else hi = mid - 1;
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
__device__ __forceinline__ float stepped(Factor f, float c, float x) {
    const float base = f.keeps ? c : x, other = f.keeps ? x : c;
    return __builtin_fmaf(f.small, other - base, base);
}
template <class T> __device__ __forceinline__ float sigmoid(float u) {
    const float s = small_sigmoid<T>(u);
    return u > 0.f ? 1.f - s : s;
}

// A workgroup's piece of a sequence: one segment (or, n == sequences, the tokens behind the last, which get zeros).
struct Piece {
    long long n, begin, end, first;   // tokens of the sequence; the sequence's first token in a packed tensor
    long long slot;
    bool last;
};
__device__ __forceinline__ bool piece_of(const Recurrence& a, long long slot, Piece& p) {
    p.slot = slot;
    p.n = sequence_of(a, slot);
    const Span span = span_of(a, p.n);
    const long long index = slot - first_slot(a, p.n, (long long)a.segment);
    p.begin = index * (long long)a.segment;
    if (index > 0 && p.begin >= span.length) return false;
    p.end = span.length - p.begin < (long long)a.segment ? span.length : p.begin + (long long)a.segment;
    p.first = span.first;
    p.last = p.end == span.length;
    return true;
}
// Where a piece's channels from c on lie at `token` of its sequence.
template <class T> __device__ __forceinline__ T* row_of(const Recurrence& a, const Rows& r, const Piece& p, long long token, unsigned c) {
    return static_cast<T*>(r.data) + (a.cu_seqlens ? (p.first + token) * r.token : p.n * r.sequence + token * r.token) + c;
}

// C neighbouring channels at a time; the last lane of an odd width has one channel in common with its neighbour, and both
// compute and write the same.
template <class T, int C> struct Few { T v[C]; };
template <class T, int C> __device__ __forceinline__ Few<T, C> load_few(const T* p) {
    Few<T, C> v;
    __builtin_memcpy(&v, __builtin_assume_aligned(p, sizeof(T)), sizeof(v));
    return v;
}
template <class T, int C> __device__ __forceinline__ void store_few(T* p, const float* v) {
    Few<T, C> r;
#pragma unroll
    for (int j = 0; j < C; ++j) r.v[j] = T(v[j]);
    __builtin_memcpy(__builtin_assume_aligned(p, sizeof(T)), &r, sizeof(r));
}
// kBatch tokens of a tensor, `step` elements apart; those that do not exist are zeros.
template <class T, int C, bool kFull> __device__ __forceinline__ void load_batch(Few<T, C> (&v)[kBatch], const T* p, ptrdiff_t step, int count) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
        if (kFull || i < count) v[i] = load_few<T, C>(p + i * step);
        else
#pragma unroll
            for (int j = 0; j < C; ++j) v[i].v[j] = T(0.f);
    }
}

constexpr int kLanes = kWave;   // a workgroup: one wave, kLanes * C channels of one piece

template <int C> __device__ __forceinline__ bool lane_channel(const Recurrence& a, unsigned block, unsigned& c) {
    c = (block * kLanes + threadIdx.x) * C;
    if (c >= a.width) return false;
    if (c + C > a.width) c = a.width - C;
    return true;
}

// What a segment makes of a state in front of it (behind it): factor * state + sum.
template <class T, int C, bool kGate, bool kBack> __global__ __launch_bounds__(kLanes) void fold_kernel(Recurrence a, unsigned blocks) {
    Piece p;
    unsigned c;
    if (!piece_of(a, blockIdx.x / blocks, p) || p.n == (long long)a.sequences || !lane_channel<C>(a, blockIdx.x % blocks, c)) return;
    float factor[C], sum[C];
#pragma unroll
    for (int j = 0; j < C; ++j) { factor[j] = 1.f; sum[j] = 0.f; }
    const auto batch = [&](long long t, auto full, int count) {
        constexpr bool kFull = decltype(full)::value;
        Few<T, C> u[kBatch], x[kBatch], g[kBatch];
        load_batch<T, C, kFull>(u, row_of<T>(a, a.forget, p, t, c), a.forget.token, count);
        load_batch<T, C, kFull>(x, kBack ? row_of<T>(a, a.dy, p, t, c) : row_of<T>(a, a.x, p, t, c), kBack ? a.dy.token : a.x.token, count);
        if constexpr (kGate && kBack) load_batch<T, C, kFull>(g, row_of<T>(a, a.gate, p, t, c), a.gate.token, count);
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int i = kBack ? kBatch - 1 - k : k;
            if (!kFull && i >= count) continue;
#pragma unroll
            for (int j = 0; j < C; ++j) {
                const Factor f = factor_of<T>(float(u[i].v[j]));
                factor[j] = kept(f, factor[j]);
                if constexpr (kBack) {
                    float d = float(x[i].v[j]);
                    if constexpr (kGate) d *= sigmoid<T>(float(g[i].v[j]));
                    sum[j] = kept(f, sum[j] + d);
                } else {
                    sum[j] = stepped(f, sum[j], float(x[i].v[j]));
                }
            }
        }
    };
    if constexpr (kBack) {
        const long long whole = (p.end - p.begin) / kBatch * kBatch + p.begin;
        if (whole < p.end) batch(whole, std::false_type(), int(p.end - whole));
        for (long long t = whole - kBatch; t >= p.begin; t -= kBatch) batch(t, std::true_type(), kBatch);
    } else {
        long long t = p.begin;
        for (; t + kBatch <= p.end; t += kBatch) batch(t, std::true_type(), kBatch);
        if (t < p.end) batch(t, std::false_type(), int(p.end - t));
    }
#pragma unroll
    for (int j = 0; j < C; ++j) a.carried[size_t(p.slot) * a.width + c + j] = float2{factor[j], sum[j]};
}

// The states in front of all segments (behind them, where kBack) from what each makes of them.
template <bool kBack> __global__ __launch_bounds__(kThreads) void join_kernel(Recurrence a) {
    const unsigned c = blockIdx.y * kThreads + threadIdx.x;
    if (c >= a.width) return;
    const long long n = blockIdx.x, first = first_slot(a, n, (long long)a.segment), length = span_of(a, n).length;
    const long long count = length > 0 ? (length + (long long)a.segment - 1) / (long long)a.segment : 1;
    const float* from = kBack ? a.d_final : a.initial;
    float s = from ? from[n * a.width + c] : 0.f;
    float2* at = a.carried + (first + (kBack ? count - 1 : 0)) * a.width + c;
    const ptrdiff_t step = kBack ? -ptrdiff_t(a.width) : ptrdiff_t(a.width);
    constexpr int kAhead = 16;
    for (long long i = 0; i < count; i += kAhead, at += kAhead * step) {
        const int m = count - i < kAhead ? int(count - i) : kAhead;
        float2 v[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (k < m) v[k] = at[k * step];
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (k < m) {
                at[k * step].x = s;
                s = __builtin_fmaf(v[k].x, s, v[k].y);
            }
    }
}

template <class T, int C, bool kGate> __global__ __launch_bounds__(kLanes) void forward_kernel(Recurrence a, unsigned blocks) {
    Piece p;
    unsigned c;
    if (!piece_of(a, blockIdx.x / blocks, p) || !lane_channel<C>(a, blockIdx.x % blocks, c)) return;
    float s[C];
#pragma unroll
    for (int j = 0; j < C; ++j) s[j] = 0.f;
    if (p.n == (long long)a.sequences) {
        for (long long t = p.begin; t < p.end; ++t) store_few<T, C>(row_of<T>(a, a.y, p, t, c), s);
        return;
    }
#pragma unroll
    for (int j = 0; j < C; ++j) {
        if (a.carried) s[j] = a.carried[size_t(p.slot) * a.width + c + j].x;
        else if (a.initial) s[j] = a.initial[p.n * a.width + c + j];
    }
    float* saved = a.saved ? a.saved + (first_slot(a, p.n, kBatch) + p.begin / kBatch) * a.width + c : nullptr;
    const auto batch = [&](long long t, auto full, int count) {
        constexpr bool kFull = decltype(full)::value;
        Few<T, C> u[kBatch], x[kBatch], g[kBatch];
        load_batch<T, C, kFull>(u, row_of<T>(a, a.forget, p, t, c), a.forget.token, count);
        load_batch<T, C, kFull>(x, row_of<T>(a, a.x, p, t, c), a.x.token, count);
        if constexpr (kGate) load_batch<T, C, kFull>(g, row_of<T>(a, a.gate, p, t, c), a.gate.token, count);
        if (saved) {
            store_few<float, C>(saved, s);
            saved += a.width;
        }
        T* y = row_of<T>(a, a.y, p, t, c);
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (!kFull && i >= count) continue;
            float o[C];
#pragma unroll
            for (int j = 0; j < C; ++j) {
                s[j] = stepped(factor_of<T>(float(u[i].v[j])), s[j], float(x[i].v[j]));
                o[j] = s[j];
                if constexpr (kGate) o[j] *= sigmoid<T>(float(g[i].v[j]));
            }
            store_few<T, C>(y + i * a.y.token, o);
        }
    };
    long long t = p.begin;
    for (; t + kBatch <= p.end; t += kBatch) batch(t, std::true_type(), kBatch);
    if (t < p.end) batch(t, std::false_type(), int(p.end - t));
    if (p.last && a.final) store_few<float, C>(a.final + p.n * a.width + c, s);
}

// From the last token to the first, G_t = sigmoid(gate_t) dy_t + f_{t+1} G_{t+1}: kBatch tokens' states again, then their gradients.
template <class T, int C, bool kGate> __global__ __launch_bounds__(kLanes) void backward_kernel(Recurrence a, unsigned blocks) {
    Piece p;
    unsigned c;
    if (!piece_of(a, blockIdx.x / blocks, p) || !lane_channel<C>(a, blockIdx.x % blocks, c)) return;
    float s[C];
#pragma unroll
    for (int j = 0; j < C; ++j) s[j] = 0.f;
    if (p.n == (long long)a.sequences) {
        const auto clear = [&](const Rows& r) {
            if (r.data)
                for (long long t = p.begin; t < p.end; ++t) store_few<T, C>(row_of<T>(a, r, p, t, c), s);
        };
        clear(a.dx);
        clear(a.dforget);
        clear(a.dgate);
        return;
    }
#pragma unroll
    for (int j = 0; j < C; ++j) {
        if (a.carried) s[j] = a.carried[size_t(p.slot) * a.width + c + j].x;
        else if (a.d_final) s[j] = a.d_final[p.n * a.width + c + j];
    }
    const float* saved = a.saved + first_slot(a, p.n, kBatch) * a.width + c;
    const auto batch = [&](long long t, auto full, int count) {
        constexpr bool kFull = decltype(full)::value;
        Few<T, C> u[kBatch], x[kBatch], d[kBatch], g[kBatch];
        load_batch<T, C, kFull>(u, row_of<T>(a, a.forget, p, t, c), a.forget.token, count);
        load_batch<T, C, kFull>(x, row_of<T>(a, a.x, p, t, c), a.x.token, count);
        load_batch<T, C, kFull>(d, row_of<T>(a, a.dy, p, t, c), a.dy.token, count);
        if constexpr (kGate) load_batch<T, C, kFull>(g, row_of<T>(a, a.gate, p, t, c), a.gate.token, count);
        const Few<float, C> before = load_few<float, C>(saved + t / kBatch * a.width);
        float state[kBatch + 1][C];
#pragma unroll
        for (int j = 0; j < C; ++j) state[0][j] = before.v[j];
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
#pragma unroll
            for (int j = 0; j < C; ++j) state[i + 1][j] = stepped(factor_of<T>(float(u[i].v[j])), state[i][j], float(x[i].v[j]));
        T* dx = a.dx.data ? row_of<T>(a, a.dx, p, t, c) : nullptr;
        T* dforget = a.dforget.data ? row_of<T>(a, a.dforget, p, t, c) : nullptr;
        T* dgate = kGate && a.dgate.data ? row_of<T>(a, a.dgate, p, t, c) : nullptr;
#pragma unroll
        for (int i = kBatch - 1; i >= 0; --i) {
            if (!kFull && i >= count) continue;
            float of_x[C], of_forget[C], of_gate[C];
#pragma unroll
            for (int j = 0; j < C; ++j) {
                const Factor f = factor_of<T>(float(u[i].v[j]));
                float dc = float(d[i].v[j]);
                if constexpr (kGate) {
                    const Factor o = factor_of<T>(float(g[i].v[j]));
                    of_gate[j] = dc * state[i + 1][j] * (o.small * (1.f - o.small));
                    dc *= keep(o);
                }
                const float total = dc + s[j];
                of_x[j] = f.keeps ? f.small * total : __builtin_fmaf(-f.small, total, total);
                of_forget[j] = total * (state[i][j] - float(x[i].v[j])) * (f.small * (1.f - f.small));
                s[j] = kept(f, total);
            }
            if (dx) store_few<T, C>(dx + i * a.dx.token, of_x);
            if (dforget) store_few<T, C>(dforget + i * a.dforget.token, of_forget);
            if constexpr (kGate)
                if (dgate) store_few<T, C>(dgate + i * a.dgate.token, of_gate);
        }
    };
    const long long whole = (p.end - p.begin) / kBatch * kBatch + p.begin;
    if (whole < p.end) batch(whole, std::false_type(), int(p.end - whole));
    for (long long t = whole - kBatch; t >= p.begin; t -= kBatch) batch(t, std::true_type(), kBatch);
    if (p.begin == 0 && a.d_initial) store_few<float, C>(a.d_initial + p.n * a.width + c, s);
}

// One token of every sequence: vectors of eight channels.
template <class T, bool kGate> __global__ __launch_bounds__(kThreads) void step_kernel(Recurrence a, unsigned vectors) {
    const size_t item = size_t(blockIdx.x) * kThreads + threadIdx.x;
    const size_t n = item / vectors, c = (item - n * vectors) * 8;
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
    return p && valid_dtype(p->dtype) && p->sequences < (size_t(1) << 31) && p->width < (size_t(1) << 31) &&
           p->tokens < (p->cu_seqlens ? size_t(1) << 31 : size_t(1) << 39);
}
size_t rows_of(const flstm_recurrence* p) { return p->cu_seqlens ? p->tokens : p->sequences * p->tokens; }
size_t slots_of(const flstm_recurrence* p, size_t size) {
    if (p->cu_seqlens) return p->tokens / size + p->sequences + 1;
    return p->sequences * (p->tokens ? ceil_div(p->tokens, size) : 1);
}
// Lanes that fill the chip.
size_t segment_of(const flstm_recurrence* p) {
    const size_t lanes = round_up(ceil_div(p->width, 2), kLanes), enough = 131072;
    if (p->sequences * lanes >= enough || p->tokens <= 128) return kWhole;
    const size_t segment = round_up(ceil_div(rows_of(p) * lanes, enough), kBatch);
    return segment < 64 ? 64 : segment;
}
size_t carried_bytes(const flstm_recurrence* p) {
    const size_t segment = segment_of(p);
    return p->tokens > segment ? slots_of(p, segment) * p->width * sizeof(float2) : 0;
}
Rows rows(const flstm_rows* r) { return r ? Rows{r->data, r->sequence, r->token} : Rows{}; }

Recurrence recurrence_of(const flstm_recurrence* p, const flstm_rows* x, const flstm_rows* forget, const flstm_rows* gate) {
    Recurrence a{};
    a.sequences = p->sequences; a.tokens = p->tokens; a.segment = segment_of(p); a.segments = slots_of(p, a.segment);
    a.cu_seqlens = p->cu_seqlens; a.width = unsigned(p->width);
    a.x = rows(x); a.forget = rows(forget); a.gate = rows(gate);
    return a;
}

// Folds the segments and joins them, where there are any, then walks.
template <bool kBack> int run(const flstm_recurrence* p, Recurrence a, void* workspace, hipStream_t stream) {
    const auto go = [&](auto zero, auto channels, auto gate) {
        typedef decltype(zero) T;
        constexpr int C = decltype(channels)::value;
        constexpr bool kGate = decltype(gate)::value;
        const size_t blocks = ceil_div(p->width, size_t(kLanes) * C), grid = a.segments * blocks;
        if (grid > kMostThreads / kLanes) return int(FLSTM_E_TOO_LARGE);
        if (carried_bytes(p) > 0) {
            a.carried = static_cast<float2*>(workspace);
            fold_kernel<T, C, kGate, kBack><<<unsigned(grid), kLanes, 0, stream>>>(a, unsigned(blocks));
            if (const int rc = launched()) return rc;
            if (p->sequences > 0) join_kernel<kBack><<<dim3(unsigned(p->sequences), unsigned(ceil_div(p->width, size_t(kThreads)))), kThreads, 0, stream>>>(a);
            if (const int rc = launched()) return rc;
        }
        if constexpr (kBack) backward_kernel<T, C, kGate><<<unsigned(grid), kLanes, 0, stream>>>(a, unsigned(blocks));
        else forward_kernel<T, C, kGate><<<unsigned(grid), kLanes, 0, stream>>>(a, unsigned(blocks));
        return launched();
    };
    return with_type(p->dtype, [&](auto zero) {
        const auto with_gate = [&](auto channels) { return a.gate.data ? go(zero, channels, std::true_type()) : go(zero, channels, std::false_type()); };
        return p->width == 1 ? with_gate(std::integral_constant<int, 1>()) : with_gate(std::integral_constant<int, 2>());
    });
}

}  // namespace
}  // namespace flstm_hip

using namespace flstm_hip;

extern "C" size_t flstm_gated_recurrence_workspace_bytes(const flstm_recurrence* p) { return valid_shape(p) ? carried_bytes(p) : 0; }
extern "C" size_t flstm_gated_recurrence_saved_rows(const flstm_recurrence* p) { return valid_shape(p) ? slots_of(p, kBatch) : 0; }

extern "C" int flstm_gated_recurrence_forward(const flstm_recurrence* p, const flstm_rows* x, const flstm_rows* forget, const flstm_rows* gate,
                                              const float* state_in, const flstm_rows* y, float* state_out, float* saved, void* workspace,
                                              void* stream) {
    if (!valid_shape(p)) return FLSTM_E_INVALID;
    if (p->width == 0 || (p->sequences == 0 && !p->cu_seqlens)) return 0;
    Recurrence a = recurrence_of(p, x, forget, gate);
    a.y = rows(y); a.initial = state_in; a.final = state_out; a.saved = saved;
    if (rows_of(p) > 0 && (!a.x.data || !a.forget.data || !a.y.data)) return FLSTM_E_INVALID;
    if (carried_bytes(p) > 0 && !workspace) return FLSTM_E_INVALID;
    return run<false>(p, a, workspace, static_cast<hipStream_t>(stream));
}

extern "C" int flstm_gated_recurrence_backward(const flstm_recurrence* p, const flstm_rows* dy, const flstm_rows* x, const flstm_rows* forget,
                                               const flstm_rows* gate, const float* saved, const float* d_state_out, const flstm_rows* dx,
                                               const flstm_rows* dforget, const flstm_rows* dgate, float* d_state_in, void* workspace, void* stream) {
    if (!valid_shape(p)) return FLSTM_E_INVALID;
    if (p->width == 0 || (p->sequences == 0 && !p->cu_seqlens)) return 0;
    Recurrence a = recurrence_of(p, x, forget, gate);
    a.dy = rows(dy); a.dx = rows(dx); a.dforget = rows(dforget); a.dgate = rows(dgate);
    a.saved = const_cast<float*>(saved); a.d_final = d_state_out; a.d_initial = d_state_in;
    if (rows_of(p) > 0 && (!a.x.data || !a.forget.data || !a.dy.data || !saved)) return FLSTM_E_INVALID;
    if ((a.dgate.data && !a.gate.data) || (carried_bytes(p) > 0 && !workspace)) return FLSTM_E_INVALID;
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
    const size_t vectors = ceil_div(p->width, 8), grid = ceil_div(p->sequences * vectors, kThreads);
    if (grid > kMostThreads / kThreads) return FLSTM_E_TOO_LARGE;
    return with_type(p->dtype, [&](auto zero) {
        typedef decltype(zero) T;
        hipStream_t s = static_cast<hipStream_t>(stream);
        if (a.gate.data) step_kernel<T, true><<<unsigned(grid), kThreads, 0, s>>>(a, unsigned(vectors));
        else step_kernel<T, false><<<unsigned(grid), kThreads, 0, s>>>(a, unsigned(vectors));
        return launched();
    });
}
