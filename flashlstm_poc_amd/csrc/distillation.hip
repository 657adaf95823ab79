// Distillation from a teacher's top logits (lm_ops.h): loss, gradient, and both in one pass.
//
// All of it is bound by reading the student's logits and writing their gradient.  A workgroup has a row.  The call that returns
// loss and gradient keeps the row in registers between the two, packed as it came, so that it is read once; the loss alone is a
// running maximum and sum; the gradient alone needs nothing but the row's saved statistics and is cut into blocks of columns.
// The teacher's entries of a row lie in LDS.  Of the columns that they name, the ones whose gradient differs from softmax, the
// values are written behind the others, each as a whole: softmax minus the sum of what all entries of that index hold, so that
// an index may come up twice, in any order, and the result is the same.
// Measured: loss and gradient of 8192 rows of 32000 bf16 logits 215 us (4.9 TB/s; a copy reaches 5.1), of 50001 388 us (4.2);
// the loss alone of 8192 rows of 50001 149 us (5.5), of 2048 rows of 32000 fp16 26 us (5.0); the gradient alone of 8192 rows of 32000
// fp16 184 us (5.7); rows of more than 65536, whose logits are read twice, 4096 of 100000 bf16, 188 + 283 us (5.2).
#include <type_traits>

#include "lm_device.h"

namespace flstm_hip {
namespace {

constexpr int kMaxTop = 1024;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLowest = -3.4028234663852886e38f;   // starts a maximum: finite, so that differences to it are numbers

struct Distill {
    size_t first, ld, ldd, d_stride;   // first: the launch's first row
    const void *logits, *teacher_logits, *teacher_index;
    void* dlogits;
    const float* d_loss;
    float* loss;
    float2* stats;        // a row's largest logit, and log2 of the sum of exp2((logit - largest) * to_log2)
    int vocabulary, top, teacher_dtype, index_64;
    float to_log2, temperature;   // differences of logits times to_log2 are exponents of two
};

__device__ __forceinline__ float max8(float8 v) {
    return fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
}
__device__ __forceinline__ float sum8(float8 v) { return ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7])); }

// log2 of a value's share where the row's largest is `most` and log2 of its sum `log_sum`.  The difference comes first: it is exact
// where it counts, and no number at all is lost in a row whose logits all lie at the lowest value of their type.
__device__ __forceinline__ float log_share(float z, float most, float log_sum, float to_log2) { return __builtin_fmaf(z - most, to_log2, -log_sum); }
__device__ __forceinline__ float8 share8(float8 z, float most, float log_sum, float to_log2) {
    float8 e;
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = __builtin_amdgcn_exp2f(log_share(z[i], most, log_sum, to_log2));
    return e;
}

// A row as its workgroup takes it: whole vectors of eight from a 16-byte boundary of `at` on, what is left in front of them with the
// first thread and what is left behind with the last.  (Rows of a vocabulary that is a multiple of nothing begin anywhere; read and
// written as they lie, 8192 of 50001 bf16 logits take 424 us instead of 388.)
struct Cut {
    int whole;        // vectors
    int head;         // elements in front of them
    int first, left;  // this thread's elements beside its vectors
};
template <class T, int THREADS> __device__ __forceinline__ Cut cut_row(const T* at, int vocabulary) {
    const int ahead = int((16 - reinterpret_cast<uintptr_t>(at) % 16) % 16 / sizeof(T));
    Cut c;
    c.head = ahead < vocabulary ? ahead : vocabulary;
    c.whole = (vocabulary - c.head) / 8;
    const int behind = c.head + c.whole * 8;
    c.first = threadIdx.x == 0 ? 0 : behind;
    c.left = threadIdx.x == 0 ? c.head : threadIdx.x == THREADS - 1 ? vocabulary - behind : 0;
    return c;
}
// This thread's elements beside its vectors, minus infinity behind them, which adds nothing to a sum.
template <class T> __device__ __forceinline__ float8 beside(const T* z, const Cut& c) {
    float8 v = load8(z + c.first, c.left);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < c.left ? v[i] : -__builtin_inff();
    return v;
}

// A pair of values over the workgroup, in all threads.
template <int THREADS, class Op> __device__ __forceinline__ float2 all_threads(float2 v, float2* scratch, Op op) {
    v.x = lanes_fold<kWave>(v.x, op);
    v.y = lanes_fold<kWave>(v.y, op);
    __syncthreads();   // (the last one's readers are done)
    if (threadIdx.x % kWave == 0) scratch[threadIdx.x / kWave] = v;
    __syncthreads();
    v = scratch[0];
#pragma unroll
    for (int w = 1; w < THREADS / kWave; ++w) {
        v.x = op(v.x, scratch[w].x);
        v.y = op(v.y, scratch[w].y);
    }
    return v;
}
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float added(float a, float b) { return a + b; }

// A row's teacher entries in LDS: index (-1: does not count), the teacher's logit and the student's.
struct Teacher {
    int index[kMaxTop];
    float weight[kMaxTop];   // the teacher's logits first, p afterwards
    float z[kMaxTop];
};

// Fills `t`; the largest of this thread's entries, kLowest without any.
template <class T, int THREADS> __device__ __forceinline__ float read_teacher(const Distill& a, size_t row, Teacher& t, bool& any) {
    float most = kLowest;
    any = false;
    for (int e = threadIdx.x; e < a.top; e += THREADS) {
        const size_t at = row * a.top + e;
        const long long index = a.index_64 ? static_cast<const long long*>(a.teacher_index)[at] : static_cast<const int*>(a.teacher_index)[at];
        const float logit = a.teacher_dtype == FLSTM_OP_F32  ? static_cast<const float*>(a.teacher_logits)[at]
                            : a.teacher_dtype == FLSTM_OP_F16 ? float(static_cast<const half_t*>(a.teacher_logits)[at])
                                                              : float(static_cast<const bfloat_t*>(a.teacher_logits)[at]);
        const bool counts = index >= 0 && index < a.vocabulary && logit != -__builtin_inff();
        t.index[e] = counts ? int(index) : -1;
        t.weight[e] = logit;
        t.z[e] = counts ? float(static_cast<const T*>(a.logits)[row * a.ld + size_t(index)]) : 0.f;
        any = any || counts;
        if (counts) most = fmaxf(most, logit);
    }
    return most;
}
// The sum of this thread's entries, relative to the largest.
template <int THREADS> __device__ __forceinline__ float teacher_mass(const Distill& a, const Teacher& t, float most) {
    float s = 0.f;
    for (int e = threadIdx.x; e < a.top; e += THREADS)
        if (t.index[e] >= 0) s += __builtin_amdgcn_exp2f(log_share(t.weight[e], most, 0.f, a.to_log2));
    return s;
}
// A distribution's largest logit and log2 of its sum.
struct Norm {
    float most, log_sum;
};
// This thread's share of sum p (log2 p - log2 q).
template <int THREADS> __device__ __forceinline__ float divergence(const Distill& a, const Teacher& t, Norm p_norm, Norm q_norm) {
    float s = 0.f;
    for (int e = threadIdx.x; e < a.top; e += THREADS) {
        if (t.index[e] < 0) continue;
        const float log_p = log_share(t.weight[e], p_norm.most, p_norm.log_sum, a.to_log2), p = __builtin_amdgcn_exp2f(log_p);
        if (p != 0.f) s += p * (log_p - log_share(t.z[e], q_norm.most, q_norm.log_sum, a.to_log2));
    }
    return s;
}
template <int THREADS> __device__ __forceinline__ void to_weights(const Distill& a, Teacher& t, Norm norm) {
    for (int e = threadIdx.x; e < a.top; e += THREADS)
        t.weight[e] = __builtin_amdgcn_exp2f(log_share(t.weight[e], norm.most, norm.log_sum, a.to_log2));
}
// The gradient at this thread's entries that lie in columns [begin, end); behind a barrier that the others' stores came before.
template <class T, int THREADS>
__device__ __forceinline__ void write_entries(const Distill& a, size_t row, const Teacher& t, float factor, Norm norm, int begin, int end) {
    T* out = static_cast<T*>(a.dlogits) + row * a.ldd;
    for (int e = threadIdx.x; e < a.top; e += THREADS) {
        const int index = t.index[e];
        if (index < begin || index >= end) continue;
        float p = 0.f;
        for (int o = 0; o < a.top; ++o)
            if (t.index[o] == index) p += t.weight[o];
        out[index] = T(factor * (__builtin_amdgcn_exp2f(log_share(t.z[e], norm.most, norm.log_sum, a.to_log2)) - p));
    }
}

// ---- the loss

template <class T, int THREADS> __global__ __launch_bounds__(THREADS) void loss_kernel(Distill a) {
    __shared__ Teacher teacher;
    __shared__ float2 scratch[THREADS / kWave];
    const size_t row = a.first + blockIdx.x;
    const T* z = static_cast<const T*>(a.logits) + row * a.ld;
    // running maximum and sum, several vectors at a time
    const Cut cut = cut_row<T, THREADS>(z, a.vocabulary);
    const float8 rest = beside(z, cut);
    float most = fmaxf(kLowest, max8(rest)), sum = sum8(share8(rest, most, 0.f, a.to_log2));
    constexpr int kAhead = 4;
    for (int base = threadIdx.x; base < cut.whole; base += kAhead * THREADS) {
        typename Vec8<T>::type v[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int i = base + j * THREADS;
            if (i < cut.whole) __builtin_memcpy(&v[j], __builtin_assume_aligned(z + cut.head + size_t(i) * 8, sizeof(T)), sizeof(v[j]));
            else v[j] = T(-__builtin_inff());
        }
        float m = most;
#pragma unroll
        for (int j = 0; j < kAhead; ++j) m = fmaxf(m, max8(__builtin_convertvector(v[j], float8)));
        sum *= __builtin_amdgcn_exp2f((most - m) * a.to_log2);
#pragma unroll
        for (int j = 0; j < kAhead; ++j) sum += sum8(share8(__builtin_convertvector(v[j], float8), m, 0.f, a.to_log2));
        most = m;
    }
    bool any;
    const float2 own{most, read_teacher<T, THREADS>(a, row, teacher, any)};
    const bool counts = __syncthreads_or(any);
    const float2 m = all_threads<THREADS>(own, scratch, larger);
    const float2 s = all_threads<THREADS>(float2{sum * __builtin_amdgcn_exp2f((most - m.x) * a.to_log2), teacher_mass<THREADS>(a, teacher, m.y)}, scratch, added);
    const Norm q_norm{m.x, __builtin_amdgcn_logf(s.x)}, p_norm{m.y, __builtin_amdgcn_logf(s.y)};
    const float2 d = all_threads<THREADS>(float2{counts ? divergence<THREADS>(a, teacher, p_norm, q_norm) : 0.f, 0.f}, scratch, added);
    if (threadIdx.x == 0) {
        a.loss[row] = counts ? a.temperature * a.temperature * kLn2 * d.x : 0.f;
        if (a.stats) a.stats[row] = float2{q_norm.most, q_norm.log_sum};
    }
}

// ---- the gradient

constexpr int kGradientThreads = 256, kGradientColumns = 16384;

template <class T> __global__ __launch_bounds__(kGradientThreads) void gradient_kernel(Distill a) {
    constexpr int THREADS = kGradientThreads;
    __shared__ Teacher teacher;
    __shared__ float2 scratch[THREADS / kWave];
    const unsigned blocks = unsigned((a.vocabulary + kGradientColumns - 1) / kGradientColumns);
    const size_t row = a.first + blockIdx.x / blocks;
    const int begin = int(blockIdx.x % blocks) * kGradientColumns;
    const int end = a.vocabulary - begin < kGradientColumns ? a.vocabulary : begin + kGradientColumns;
    const T* z = static_cast<const T*>(a.logits) + row * a.ld;
    T* out = static_cast<T*>(a.dlogits) + row * a.ldd;
    bool any;
    const float most = read_teacher<T, THREADS>(a, row, teacher, any);
    if (!__syncthreads_or(any)) {
        for (int c = begin + int(threadIdx.x) * 8; c < end; c += THREADS * 8) {
            const float8 zero = 0.f;
            store8(out + c, zero, end - c);
        }
        return;
    }
    const float m = all_threads<THREADS>(float2{most, 0.f}, scratch, larger).x;
    const float mass = all_threads<THREADS>(float2{teacher_mass<THREADS>(a, teacher, m), 0.f}, scratch, added).x;
    to_weights<THREADS>(a, teacher, Norm{m, __builtin_amdgcn_logf(mass)});
    const Norm norm{a.stats[row].x, a.stats[row].y};
    const float factor = a.d_loss[row * a.d_stride] * a.temperature;
    const Cut cut = cut_row<T, THREADS>(out + begin, end - begin);
    z += begin;
    out += begin;
    for (int i = threadIdx.x; i < cut.whole; i += THREADS) {
        const size_t c = cut.head + size_t(i) * 8;
        store8(out + c, factor * share8(load8(z + c), norm.most, norm.log_sum, a.to_log2));
    }
    store8(out + cut.first, factor * share8(beside(z, cut), norm.most, norm.log_sum, a.to_log2), cut.left);
    __syncthreads();
    write_entries<T, THREADS>(a, row, teacher, factor, norm, begin, end);
}

// ---- both

// A row in the registers of its workgroup: R vectors of eight values a thread.
template <class T, int THREADS, int R> __global__ __launch_bounds__(THREADS) void train_kernel(Distill a) {
    __shared__ Teacher teacher;
    __shared__ float2 scratch[THREADS / kWave];
    const size_t row = a.first + blockIdx.x;
    const T* z = static_cast<const T*>(a.logits) + row * a.ld;
    T* out = static_cast<T*>(a.dlogits) + row * a.ldd;
    typedef typename Vec8<T>::type vec;
    const int tid = threadIdx.x;
    const Cut cut = cut_row<T, THREADS>(out, a.vocabulary);
    vec v[R + 1];
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const int i = j * THREADS + tid;
        if (i < cut.whole) __builtin_memcpy(&v[j], __builtin_assume_aligned(z + cut.head + size_t(i) * 8, sizeof(T)), sizeof(vec));
        else v[j] = T(-__builtin_inff());
    }
    v[R] = __builtin_convertvector(beside(z, cut), vec);
    // (Between the three readings the row is hidden from the compiler, which would otherwise keep it converted, in twice the registers.)
    const auto hide = [&] {
#pragma unroll
        for (int j = 0; j <= R; ++j) asm volatile("" : "+v"(v[j]));
    };
    bool any;
    const float teacher_most = read_teacher<T, THREADS>(a, row, teacher, any);
    const bool counts = __syncthreads_or(any);
    float most = kLowest;
    hide();
#pragma unroll
    for (int j = 0; j <= R; ++j) most = fmaxf(most, max8(__builtin_convertvector(v[j], float8)));
    const float2 m = all_threads<THREADS>(float2{most, teacher_most}, scratch, larger);
    float sum = 0.f;
    hide();
#pragma unroll
    for (int j = 0; j <= R; ++j) sum += sum8(share8(__builtin_convertvector(v[j], float8), m.x, 0.f, a.to_log2));
    const float2 s = all_threads<THREADS>(float2{sum, teacher_mass<THREADS>(a, teacher, m.y)}, scratch, added);
    const Norm q_norm{m.x, __builtin_amdgcn_logf(s.x)}, p_norm{m.y, __builtin_amdgcn_logf(s.y)};
    const float2 d = all_threads<THREADS>(float2{counts ? divergence<THREADS>(a, teacher, p_norm, q_norm) : 0.f, 0.f}, scratch, added);
    if (tid == 0) a.loss[row] = counts ? a.temperature * a.temperature * kLn2 * d.x : 0.f;
    const float factor = a.d_loss[row * a.d_stride] * a.temperature;
    hide();
#pragma unroll
    for (int j = 0; j <= R; ++j) {
        const int i = j * THREADS + tid;
        float8 g = 0.f;
        if (counts) g = factor * share8(__builtin_convertvector(v[j], float8), q_norm.most, q_norm.log_sum, a.to_log2);
        if (j == R) store8(out + cut.first, g, cut.left);
        else if (i < cut.whole) store8(out + cut.head + size_t(i) * 8, g);
    }
    if (!counts) return;
    to_weights<THREADS>(a, teacher, p_norm);
    __syncthreads();
    write_entries<T, THREADS>(a, row, teacher, factor, q_norm, 0, a.vocabulary);
}

// ---- host side

bool valid_problem(const flstm_distillation* p) {
    return p && valid_dtype(p->dtype) && valid_dtype(p->teacher_dtype) && p->top >= 1 && p->top <= kMaxTop && p->temperature > 0.f &&
           p->temperature < __builtin_inff() && kLog2e / p->temperature < __builtin_inff() && p->vocabulary >= 1 && p->vocabulary < (size_t(1) << 31) - 65536 && p->ld >= p->vocabulary &&
           p->rows < (size_t(1) << 31) && (p->rows == 0 || (p->logits && p->teacher_logits && p->teacher_index));
}

Distill distill_of(const flstm_distillation* p) {
    Distill a{};
    a.ld = p->ld; a.logits = p->logits; a.teacher_logits = p->teacher_logits; a.teacher_index = p->teacher_index;
    a.vocabulary = int(p->vocabulary); a.top = p->top; a.teacher_dtype = p->teacher_dtype; a.index_64 = p->index_64;
    a.temperature = p->temperature; a.to_log2 = kLog2e / p->temperature;
    return a;
}

// The most that a row in registers may have: 16 vectors of eight 16-bit values a thread of 512, or eight of fp32 a thread of 1024.
// Two workgroups of 512 threads fit a CU, so that one's row arrives while the other's gradient leaves: 8192 rows of 50048 bf16
// logits take 366 us (4.5 TB/s), where one of 1024 threads took 472.  (100000 of them with 16 vectors a thread of 1024, alone on
// its CU, took 457 us for 4096 rows: no less than the two passes that read the logits twice.)  Up to 16384 logits a row the same holds for
// smaller workgroups: 8192 rows of 12000 bf16 logits take 85 us with 256 threads of eight vectors, 103 with 512 of four, 165 with 1024
// of two; 32 rows 8.8, 8.6 and 9.3.
constexpr size_t kHeld = 65536;

// Launches `go(problem, rows)` for so many rows at a time that a launch stays below its limit of 2^32 threads: of at most 1024 for
// each of `workgroups` a row.
template <class F> int in_launches(Distill a, size_t rows, size_t workgroups, F&& go) {
    const size_t most = (size_t(1) << 21) / workgroups;
    for (a.first = 0; a.first < rows; a.first += most)
        if (const int rc = go(a, unsigned(rows - a.first < most ? rows - a.first : most))) return rc;
    return 0;
}

}  // namespace
}  // namespace flstm_hip

using namespace flstm_hip;

extern "C" int flstm_distillation_forward(const flstm_distillation* p, float* loss, float* stats, void* stream) {
    if (!valid_problem(p) || (p->rows > 0 && !loss)) return FLSTM_E_INVALID;
    if (p->rows == 0) return 0;
    Distill a = distill_of(p);
    a.loss = loss; a.stats = reinterpret_cast<float2*>(stats);
    return with_type(p->dtype, [&](auto zero) {
        typedef decltype(zero) T;
        // (256 threads a row where the rows fill the chip, so that eight of them are under way in a CU: 1024 rows of 32000 bf16 16 us
        // instead of 20, 2048 of fp16 26 instead of 35; 1024 threads where they do not and a row is long: 64 rows of 32000 bf16 6.8 us instead
        // of 9.4, of 8192 6.1 where 256 threads take 4.9.)
        return in_launches(a, p->rows, 1, [&](const Distill& part, unsigned rows) {
            if (p->vocabulary <= 8192 || p->rows >= 256) loss_kernel<T, 256><<<rows, 256, 0, static_cast<hipStream_t>(stream)>>>(part);
            else loss_kernel<T, 1024><<<rows, 1024, 0, static_cast<hipStream_t>(stream)>>>(part);
            return launched();
        });
    });
}

extern "C" int flstm_distillation_backward(const flstm_distillation* p, const float* stats, const float* d_loss, size_t d_stride,
                                           void* dlogits, size_t ldd, void* stream) {
    if (!valid_problem(p) || (p->rows > 0 && (!stats || !d_loss || !dlogits)) || ldd < p->vocabulary) return FLSTM_E_INVALID;
    if (p->rows == 0) return 0;
    Distill a = distill_of(p);
    a.stats = reinterpret_cast<float2*>(const_cast<float*>(stats)); a.d_loss = d_loss; a.d_stride = d_stride; a.dlogits = dlogits; a.ldd = ldd;
    const unsigned blocks = unsigned(ceil_div(p->vocabulary, size_t(kGradientColumns)));
    return with_type(p->dtype, [&](auto zero) {
        return in_launches(a, p->rows, blocks, [&](const Distill& part, unsigned rows) {
            gradient_kernel<decltype(zero)><<<rows * blocks, kGradientThreads, 0, static_cast<hipStream_t>(stream)>>>(part);
            return launched();
        });
    });
}

extern "C" size_t flstm_distillation_workspace_bytes(const flstm_distillation* p) {
    return valid_problem(p) && p->vocabulary > kHeld ? round_up(p->rows * 2 * sizeof(float), 16) : 0;
}

extern "C" int flstm_distillation_train(const flstm_distillation* p, const float* d_loss, size_t d_stride, float* loss, void* dlogits,
                                        size_t ldd, void* workspace, void* stream) {
    if (!valid_problem(p) || (p->rows > 0 && (!loss || !d_loss || !dlogits)) || ldd < p->vocabulary) return FLSTM_E_INVALID;
    if (p->rows == 0) return 0;
    if (p->vocabulary > kHeld) {   // one pass behind the other, the rows' statistics in the workspace
        if (!workspace) return FLSTM_E_INVALID;
        const int rc = flstm_distillation_forward(p, loss, static_cast<float*>(workspace), stream);
        return rc != 0 ? rc : flstm_distillation_backward(p, static_cast<const float*>(workspace), d_loss, d_stride, dlogits, ldd, stream);
    }
    Distill a = distill_of(p);
    a.loss = loss; a.d_loss = d_loss; a.d_stride = d_stride; a.dlogits = dlogits; a.ldd = ldd;
    return with_type(p->dtype, [&](auto zero) {
        typedef decltype(zero) T;
        const auto go = [&](auto threads, auto vectors) {
            return in_launches(a, p->rows, 1, [&](const Distill& part, unsigned rows) {
                train_kernel<T, decltype(threads)::value, decltype(vectors)::value><<<rows, threads.value, 0, static_cast<hipStream_t>(stream)>>>(part);
                return launched();
            });
        };
        const std::integral_constant<int, 256> few;
        const std::integral_constant<int, 512> some;
        const std::integral_constant<int, 1024> many;
        if (p->vocabulary <= 2048) return go(few, std::integral_constant<int, 1>());
        if (p->vocabulary <= 8192) return go(few, std::integral_constant<int, 4>());
        if (p->vocabulary <= 16384) return go(few, std::integral_constant<int, 8>());
        if (p->vocabulary <= 32768) return go(some, std::integral_constant<int, 8>());
        if constexpr (sizeof(T) == 2) return go(some, std::integral_constant<int, 16>());
        else return go(many, std::integral_constant<int, 8>());
    });
}
