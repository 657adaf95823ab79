// Layer norm on a residual stream, forward and backward (lm_ops.h).
//
// Both passes are bound by memory: forward reads x and the residual and writes total and y, backward reads dy, total and
// d_total and writes dx, a few operations a value.  A row therefore stays in registers from its one load to its store: L lanes
// of a wave (or a whole workgroup, for rows of more than 2048) hold V vectors of eight values each.  The variance is summed over
// the centred values, not as a difference of two moments, which costs a second reduction and no traffic.
// Measured on 262144 rows of 1024 fp16 values with a residual, under the profiler: forward 397 us, 5.4 TB/s; backward with the parameters'
// gradients 404 + 5 us, 5.3 TB/s (a copy reaches 5.1).  32 such rows take 4.3 us forward, a launch and two trips to memory.
#include "lm_device.h"

namespace flstm_hip {
namespace {

constexpr int kNormThreads = 256;
constexpr size_t kMaxWidth = 16384;
constexpr size_t kMaxPartials = 1024;   // workgroups of a backward pass, each with a row of partial sums of dweight and dbias

struct NormForward {
    size_t rows;
    int width;
    const void *x, *residual;
    size_t ldx, ldr;
    const float *weight, *bias;
    float eps;
    void *total, *y;
    float *mean, *rstd;
};

struct NormBackward {
    size_t rows;
    int width;
    const void *dy, *total, *d_total;
    size_t lddy, ldt, lddt;
    const float *weight, *mean, *rstd;
    void* dx;
    float* partials;   // [workgroup][dweight, dbias][width], or null
};

// Sum over the L lanes that hold a row, in all of them.  `scratch`: a float per wave, used where L is more than a wave.
template <int L> __device__ __forceinline__ float row_sum(float v, float* scratch) {
    if constexpr (L <= kWave) {
        return lanes_sum<L>(v);
    } else {
        v = lanes_sum<kWave>(v);
        __syncthreads();   // (the last sum's readers are done)
        if (threadIdx.x % kWave == 0) scratch[threadIdx.x / kWave] = v;
        __syncthreads();
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < L / kWave; ++w) s += scratch[w];
        return s;
    }
}

__device__ __forceinline__ float sum8(float8 v) {
    return ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
}

// Zero behind a row's end.
__device__ __forceinline__ float8 keep8(float8 v, int n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? v[i] : 0.f;
    return v;
}

__device__ __forceinline__ float8 ones8() { float8 v = 1.f; return v; }

template <class T, int L, int V>
__global__ __launch_bounds__(L > kNormThreads ? L : kNormThreads) void norm_forward_kernel(NormForward a) {
    constexpr int kThreads = L > kNormThreads ? L : kNormThreads, kRows = kThreads / L;
    __shared__ float scratch[kThreads / kWave];
    const int lane = threadIdx.x % L;
    const float count = float(a.width);   // (divided by, not multiplied with its reciprocal: a row of one value has that mean exactly)
    for (size_t row = size_t(blockIdx.x) * kRows + threadIdx.x / L; row < a.rows; row += size_t(gridDim.x) * kRows) {
        const T* x = static_cast<const T*>(a.x) + row * a.ldx;
        float8 v[V];
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (j * L + lane) * 8;
            v[j] = load8(x + c, a.width - c);
        }
        if (a.residual) {
            const T* r = static_cast<const T*>(a.residual) + row * a.ldr;
            T* t = static_cast<T*>(a.total) + row * a.width;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int c = (j * L + lane) * 8;
                v[j] += load8(r + c, a.width - c);
                // the norm reads the stream as the backward pass will find it: in the tensors' type
                v[j] = __builtin_convertvector(__builtin_convertvector(v[j], typename Vec8<T>::type), float8);
                store8(t + c, v[j], a.width - c);
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) s += sum8(v[j]);
        const float mean = row_sum<L>(s, scratch) / count;
        s = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            v[j] = keep8(v[j] - mean, a.width - (j * L + lane) * 8);
            s += sum8(v[j] * v[j]);
        }
        const float rstd = rsqrtf(row_sum<L>(s, scratch) / count + a.eps);
        T* y = static_cast<T*>(a.y) + row * a.width;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (j * L + lane) * 8, n = a.width - c;
            const float8 w = a.weight ? load8(a.weight + c, n) : ones8();
            float8 o = v[j] * rstd * w;
            if (a.bias) o += load8(a.bias + c, n);
            store8(y + c, o, n);
        }
        if (lane == 0) {
            if (a.mean) a.mean[row] = mean;
            if (a.rstd) a.rstd[row] = rstd;
        }
    }
}

// The sums over rows: every lane keeps those of its own columns in registers over all rows that its workgroup takes, the
// workgroup adds up its rows' shares and leaves one row of partial sums, and norm_reduce_kernel adds those up.  No atomics: the
// order depends on the sizes alone.
template <class T, int L, int V, bool kParameters>
__global__ __launch_bounds__(L > kNormThreads ? L : kNormThreads) void norm_backward_kernel(NormBackward a) {
    constexpr int kThreads = L > kNormThreads ? L : kNormThreads, kRows = kThreads / L;
    __shared__ float scratch[kThreads / kWave];
    __shared__ float8 share[kParameters && kRows > 1 ? kThreads : 1];
    const int lane = threadIdx.x % L;
    const float inverse = 1.f / float(a.width);
    // (512 lanes with four vectors would need more than their 256 registers: they read the weight for every row, from the caches)
    constexpr bool kKeepWeight = L <= kNormThreads;
    const auto weight = [&](int c) { return a.weight ? load8(a.weight + c, a.width - c) : ones8(); };
    float8 w[kKeepWeight ? V : 1], dw[V], db[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if constexpr (kKeepWeight) w[j] = weight((j * L + lane) * 8);
        dw[j] = db[j] = 0.f;
    }
    for (size_t row = size_t(blockIdx.x) * kRows + threadIdx.x / L; row < a.rows; row += size_t(gridDim.x) * kRows) {
        const T *dy = static_cast<const T*>(a.dy) + row * a.lddy, *total = static_cast<const T*>(a.total) + row * a.ldt;
        int at = threadIdx.x % L;
        asm volatile("" : "+v"(at));   // (columns and addresses are formed for every row: kept, they take registers)
        const T* dt = a.d_total ? static_cast<const T*>(a.d_total) + row * a.lddt : nullptr;
        const float mean = a.mean[row], rstd = a.rstd[row];
        float8 h[V], n[V];
        typename Vec8<T>::type more[V];   // of d_total, as it came: requested with the others, used at the end
        float sh = 0.f, shn = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (j * L + at) * 8;
            h[j] = load8(dy + c, a.width - c);
            n[j] = load8(total + c, a.width - c);
            more[j] = T(0.f);
            if (dt) more[j] = __builtin_convertvector(load8(dt + c, a.width - c), typename Vec8<T>::type);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            n[j] = keep8((n[j] - mean) * rstd, a.width - (j * L + at) * 8);
            if constexpr (kParameters) {
                dw[j] += h[j] * n[j];
                db[j] += h[j];
            }
            if constexpr (!kKeepWeight) w[0] = weight((j * L + at) * 8);
            h[j] *= w[kKeepWeight ? j : 0];
            sh += sum8(h[j]);
            shn += sum8(h[j] * n[j]);
        }
        const float mh = row_sum<L>(sh, scratch) * inverse, mhn = row_sum<L>(shn, scratch) * inverse;
        T* dx = static_cast<T*>(a.dx) + row * a.width;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = (j * L + at) * 8;
            store8(dx + c, rstd * (h[j] - mh - n[j] * mhn) + __builtin_convertvector(more[j], float8), a.width - c);
        }
    }
    if constexpr (kParameters) {
        float* out = a.partials + size_t(blockIdx.x) * 2 * a.width;
#pragma unroll
        for (int j = 0; j < V; ++j) {
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                float8 s = which ? db[j] : dw[j];
                if constexpr (kRows > 1) {
                    __syncthreads();
                    share[threadIdx.x] = s;
                    __syncthreads();
                    if (threadIdx.x >= L) continue;
                    s = share[lane];
#pragma unroll 1
                    for (int r = 1; r < kRows; ++r) s += share[r * L + lane];
                }
                const int c = (j * L + lane) * 8;
                store8(out + size_t(which) * a.width + c, s, a.width - c);
            }
        }
    }
}

// 32 columns by 32 groups of partial rows a workgroup.
__global__ __launch_bounds__(1024) void norm_reduce_kernel(const float* partials, int count, int width, float* dweight, float* dbias) {
    __shared__ float share[32][33];
    float* out = blockIdx.y ? dbias : dweight;
    if (!out) return;
    const int x = threadIdx.x % 32, group = threadIdx.x / 32, c = blockIdx.x * 32 + x;
    float s = 0.f;
    if (c < width) {
        const float* p = partials + size_t(blockIdx.y) * width + c;
#pragma unroll 8
        for (int i = group; i < count; i += 32) s += p[size_t(i) * 2 * width];
    }
    share[group][x] = s;
    __syncthreads();
    if (group == 0 && c < width) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) t += share[i][x];
        out[c] = t;
    }
}

// Calls `f` with the lanes and vectors that hold a row of this width.
template <int L, int V> struct Hold {
    static constexpr int lanes = L, vectors = V;
};
template <class F> int with_hold(size_t width, F&& f) {
    if (width <= 64) return f(Hold<8, 1>());
    if (width <= 128) return f(Hold<16, 1>());
    if (width <= 256) return f(Hold<32, 1>());
    if (width <= 512) return f(Hold<64, 1>());
    if (width <= 1024) return f(Hold<64, 2>());
    if (width <= 2048) return f(Hold<64, 4>());
    if (width <= 4096) return f(Hold<256, 2>());
    if (width <= 8192) return f(Hold<256, 4>());
    return f(Hold<512, 4>());
}

int rows_per_workgroup(size_t width) {
    return with_hold(width, [](auto hold) { return hold.lanes > kNormThreads ? 1 : kNormThreads / hold.lanes; });
}

// Workgroups of a backward pass: at least four turns each where there are many rows, so that the partial sums stay small
// against the rows.
size_t backward_workgroups(size_t rows, size_t width) {
    const size_t n = ceil_div(rows, size_t(rows_per_workgroup(width)) * 4);
    return n < kMaxPartials ? n : kMaxPartials;
}

}  // namespace
}  // namespace flstm_hip

using namespace flstm_hip;

extern "C" int flstm_layer_norm_forward(size_t rows, size_t width, const void* x, size_t ldx, const void* residual, size_t ldr,
                                        flstm_op_dtype dtype, const float* weight, const float* bias, float eps, void* total,
                                        void* y, float* mean, float* rstd, void* stream) {
    if (!valid_dtype(dtype) || !(eps >= 0.f)) return FLSTM_E_INVALID;
    if (rows == 0 || width == 0) return 0;
    if (width > kMaxWidth) return FLSTM_E_TOO_LARGE;
    if (!x || !y || (residual && !total)) return FLSTM_E_INVALID;
    const NormForward a{rows, int(width), x, residual, ldx, ldr, weight, bias, eps, total, y, mean, rstd};
    return with_type(dtype, [&](auto zero) {
        return with_hold(width, [&](auto hold) {
            constexpr int L = decltype(hold)::lanes, V = decltype(hold)::vectors, threads = L > kNormThreads ? L : kNormThreads;
            const size_t wanted = ceil_div(rows, size_t(threads / L));
            const unsigned grid = unsigned(wanted < (1u << 20) ? wanted : (1u << 20));
            norm_forward_kernel<decltype(zero), L, V><<<grid, threads, 0, static_cast<hipStream_t>(stream)>>>(a);
            return launched();
        });
    });
}

extern "C" size_t flstm_layer_norm_workspace_bytes(size_t rows, size_t width) {
    if (rows == 0 || width == 0 || width > kMaxWidth) return 0;
    return backward_workgroups(rows, width) * 2 * width * sizeof(float);
}

extern "C" int flstm_layer_norm_backward(size_t rows, size_t width, const void* dy, size_t lddy, const void* total, size_t ldt,
                                         const void* d_total, size_t lddt, flstm_op_dtype dtype, const float* weight,
                                         const float* mean, const float* rstd, void* dx, float* dweight, float* dbias,
                                         void* workspace, void* stream) {
    if (!valid_dtype(dtype)) return FLSTM_E_INVALID;
    if (width > kMaxWidth) return FLSTM_E_TOO_LARGE;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool parameters = dweight || dbias;
    if (width == 0) return 0;
    if (rows && (!dy || !total || !mean || !rstd || !dx || (parameters && !workspace))) return FLSTM_E_INVALID;
    const size_t count = rows ? backward_workgroups(rows, width) : 0;
    if (rows) {
        const NormBackward a{rows, int(width), dy, total, d_total, lddy, ldt, lddt, weight, mean, rstd, dx, static_cast<float*>(workspace)};
        const int rc = with_type(dtype, [&](auto zero) {
            return with_hold(width, [&](auto hold) {
                constexpr int L = decltype(hold)::lanes, V = decltype(hold)::vectors, threads = L > kNormThreads ? L : kNormThreads;
                if (parameters) norm_backward_kernel<decltype(zero), L, V, true><<<unsigned(count), threads, 0, s>>>(a);
                else norm_backward_kernel<decltype(zero), L, V, false><<<unsigned(count), threads, 0, s>>>(a);
                return launched();
            });
        });
        if (rc != 0) return rc;
    }
    if (parameters) {   // (of no rows: zeros)
        norm_reduce_kernel<<<dim3(unsigned(ceil_div(width, 32)), 2), 1024, 0, s>>>(static_cast<const float*>(workspace), int(count),
                                                                                  int(width), dweight, dbias);
        return launched();
    }
    return 0;
}
