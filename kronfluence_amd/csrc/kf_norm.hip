// kf_norm.hip -- layer norm and RMS norm over the last axis, forward and backward (see include/kronfluence_hip.h, "Model passes").
//
//     mu = mean x (layer norm; 0 for RMS norm)     r = 1 / sqrt(mean (x - mu)^2 + eps)     xhat = (x - mu) r     y = xhat w + b
//     u = g w      dx = r (u - mean u - xhat mean(u xhat))   (no mean u for RMS norm)      dw = sum_rows g xhat     db = sum_rows g
//
// Bound by memory: a row is read once, held in registers as fp32 (the variance is a second pass over the REGISTERS, so it does not
// cancel), and written once.  A group of LANES lanes owns a row: one wave up to 2 048 columns (no barrier at all), eight waves up to
// 16 384, beyond that the row is re-read from the cache.  The weight's gradient needs no atomics: a group adds up the columns of its
// rows in registers, each workgroup writes one partial row, and a second kernel adds the partial rows in a fixed order.
// All arithmetic is fp32; the outputs are rounded once.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/kronfluence_hip.h"

namespace {

constexpr int THREADS = 256, WIDE_THREADS = 512;
constexpr int VEC = 8;                       // columns per chunk
constexpr int WAVE_MAX = 64 * VEC * 4;       // columns a wave holds in registers
constexpr int WIDE_MAX = WIDE_THREADS * VEC * 4;

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int launch_status() { return hipGetLastError() == hipSuccess ? KF_OK : KF_ERR_LAUNCH_FAILED; }

// Eight consecutive elements at any element-aligned address (rows of odd widths start anywhere).
template <class T>
struct __attribute__((packed, aligned(sizeof(T)))) Chunk { T v[VEC]; };

template <class T>
__device__ __forceinline__ void load8(float (&x)[VEC], const T* p, int64_t column, int64_t width) {
    if (column + VEC <= width) {
        const Chunk<T> c = *reinterpret_cast<const Chunk<T>*>(p + column);
#pragma unroll
        for (int i = 0; i < VEC; ++i) x[i] = static_cast<float>(c.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) x[i] = column + i < width ? static_cast<float>(p[column + i]) : 0.0f;
    }
}

template <class T>
__device__ __forceinline__ void store8(T* p, int64_t column, int64_t width, const float (&x)[VEC]) {
    if (column + VEC <= width) {
        Chunk<T> c;
#pragma unroll
        for (int i = 0; i < VEC; ++i) c.v[i] = static_cast<T>(x[i]);
        *reinterpret_cast<Chunk<T>*>(p + column) = c;
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (column + i < width) p[column + i] = static_cast<T>(x[i]);
    }
}

// eight elements of a vector whose type is known at run time only (weight, bias: read once per workgroup)
__device__ __forceinline__ void load8_as(float (&x)[VEC], const void* p, int dtype, int64_t column, int64_t width) {
    if (dtype == KF_F32) load8(x, reinterpret_cast<const float*>(p), column, width);
    else if (dtype == KF_BF16) load8(x, reinterpret_cast<const __bf16*>(p), column, width);
    else load8(x, reinterpret_cast<const _Float16*>(p), column, width);
}

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) x += __shfl_xor(x, m);
    return x;
}

// Sums over the LANES lanes of a row's group; `scratch` is used by groups of several waves (two barriers).
template <int LANES>
__device__ __forceinline__ float group_sum(float x, float* scratch) {
    x = wave_sum(x);
    if constexpr (LANES > 64) {
        const int wave = threadIdx.x >> 6;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) scratch[wave] = x;
        __syncthreads();
        x = 0.0f;
#pragma unroll
        for (int i = 0; i < LANES / 64; ++i) x += scratch[i];
    }
    return x;
}
template <int LANES>
__device__ __forceinline__ void group_sum2(float& x, float& y, float* scratch) {
    x = wave_sum(x);
    y = wave_sum(y);
    if constexpr (LANES > 64) {
        const int wave = threadIdx.x >> 6;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) { scratch[2 * wave] = x; scratch[2 * wave + 1] = y; }
        __syncthreads();
        x = y = 0.0f;
#pragma unroll
        for (int i = 0; i < LANES / 64; ++i) { x += scratch[2 * i]; y += scratch[2 * i + 1]; }
    }
}

struct ForwardArgs {
    void* y;
    float* stats;         // [rows][2]: mu, r; or null
    const void *x, *weight, *bias;
    int64_t rows, width, ld;   // ld: elements between rows of x
    int w_dtype, centred;
    float eps;
};

// LANES lanes per row, NV chunks per lane: width <= LANES * NV * VEC.  The weights stay in registers for the workgroup's rows.
template <class X, class Y, int LANES, int NV>
__global__ __launch_bounds__(LANES > 64 ? LANES : THREADS) void norm_forward_kernel(const ForwardArgs a) {
    constexpr int BLOCK = LANES > 64 ? LANES : THREADS, GROUPS = BLOCK / LANES;
    __shared__ float scratch[16];
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    const float inv = 1.0f / static_cast<float>(a.width);
    float w[NV][VEC], b[NV][VEC];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int64_t c = (lane + j * LANES) * VEC;
#pragma unroll
        for (int i = 0; i < VEC; ++i) { w[j][i] = 1.0f; b[j][i] = 0.0f; }
        if (a.weight) load8_as(w[j], a.weight, a.w_dtype, c, a.width);
        if (a.bias) load8_as(b[j], a.bias, a.w_dtype, c, a.width);
    }
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * GROUPS + group; row < a.rows; row += static_cast<int64_t>(gridDim.x) * GROUPS) {
        const X* x = reinterpret_cast<const X*>(a.x) + row * a.ld;
        float v[NV][VEC];
#pragma unroll
        for (int j = 0; j < NV; ++j) load8(v[j], x, (lane + j * LANES) * VEC, a.width);
        float mu = 0.0f;
        if (a.centred) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < VEC; ++i) mu += v[j][i];
            mu = group_sum<LANES>(mu, scratch) * inv;
        }
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                v[j][i] = (lane + j * LANES) * VEC + i < a.width ? v[j][i] - mu : 0.0f;
                ss = fmaf(v[j][i], v[j][i], ss);
            }
        const float r = 1.0f / sqrtf(group_sum<LANES>(ss, scratch) * inv + a.eps);
        Y* y = reinterpret_cast<Y*>(a.y) + row * a.width;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float out[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) out[i] = fmaf(v[j][i] * r, w[j][i], b[j][i]);
            const int64_t c = (lane + j * LANES) * VEC;
            if (c < a.width) store8(y, c, a.width, out);
        }
        if (a.stats && lane == 0) { a.stats[2 * row] = mu; a.stats[2 * row + 1] = r; }
    }
}

// Rows wider than the registers: the row is read three times (from memory once, then from the cache).
template <class X, class Y>
__global__ __launch_bounds__(WIDE_THREADS) void norm_forward_long_kernel(const ForwardArgs a) {
    __shared__ float scratch[16];
    const float inv = 1.0f / static_cast<float>(a.width);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const X* x = reinterpret_cast<const X*>(a.x) + row * a.ld;
        float mu = 0.0f, ss = 0.0f, v[VEC], w[VEC], b[VEC];
        if (a.centred) {
            for (int64_t c = threadIdx.x * VEC; c < a.width; c += WIDE_THREADS * VEC) {
                load8(v, x, c, a.width);
#pragma unroll
                for (int i = 0; i < VEC; ++i) mu += v[i];
            }
            mu = group_sum<WIDE_THREADS>(mu, scratch) * inv;
        }
        for (int64_t c = threadIdx.x * VEC; c < a.width; c += WIDE_THREADS * VEC) {
            load8(v, x, c, a.width);
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (c + i < a.width) ss = fmaf(v[i] - mu, v[i] - mu, ss);
        }
        const float r = 1.0f / sqrtf(group_sum<WIDE_THREADS>(ss, scratch) * inv + a.eps);
        Y* y = reinterpret_cast<Y*>(a.y) + row * a.width;
        for (int64_t c = threadIdx.x * VEC; c < a.width; c += WIDE_THREADS * VEC) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) { w[i] = 1.0f; b[i] = 0.0f; }
            if (a.weight) load8_as(w, a.weight, a.w_dtype, c, a.width);
            if (a.bias) load8_as(b, a.bias, a.w_dtype, c, a.width);
            load8(v, x, c, a.width);
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[i] = fmaf((v[i] - mu) * r, w[i], b[i]);
            store8(y, c, a.width, v);
        }
        if (a.stats && threadIdx.x == 0) { a.stats[2 * row] = mu; a.stats[2 * row + 1] = r; }
    }
}

struct BackwardArgs {
    void* dx;             // or null
    float* partial;       // [workgroups][1 or 2][width]: sums of g xhat, then of g; or null
    const float* stats;
    const void *g, *x, *weight;
    int64_t rows, width, ld;
    int w_dtype, centred, with_bias;
};

// As the forward kernel; every group adds up the columns of its rows for dw and db beside writing dx.
template <class X, class G, int LANES, int NV>
__global__ __launch_bounds__(LANES > 64 ? LANES : THREADS) void norm_backward_kernel(const BackwardArgs a) {
    constexpr int BLOCK = LANES > 64 ? LANES : THREADS, GROUPS = BLOCK / LANES, COLUMNS = LANES * NV * VEC;
    __shared__ float scratch[16];
    __shared__ float joined[GROUPS > 1 ? COLUMNS : 1];
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    const float inv = 1.0f / static_cast<float>(a.width);
    float w[NV][VEC], dw[NV][VEC], db[NV][VEC];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) { w[j][i] = 1.0f; dw[j][i] = 0.0f; db[j][i] = 0.0f; }
        if (a.weight) load8_as(w[j], a.weight, a.w_dtype, (lane + j * LANES) * VEC, a.width);
    }
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * GROUPS + group; row < a.rows; row += static_cast<int64_t>(gridDim.x) * GROUPS) {
        const X* x = reinterpret_cast<const X*>(a.x) + row * a.ld;
        const G* g = reinterpret_cast<const G*>(a.g) + row * a.width;
        const float mu = a.stats[2 * row], r = a.stats[2 * row + 1];
        float h[NV][VEC], u[NV][VEC], mean_u = 0.0f, mean_uh = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t c = (lane + j * LANES) * VEC;
            load8(h[j], x, c, a.width);
            load8(u[j], g, c, a.width);
        }
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                h[j][i] = (h[j][i] - mu) * r;    // (columns behind the width: g is 0 there)
                dw[j][i] = fmaf(u[j][i], h[j][i], dw[j][i]);
                db[j][i] += u[j][i];
                u[j][i] *= w[j][i];
                mean_u += u[j][i];
                mean_uh = fmaf(u[j][i], h[j][i], mean_uh);
            }
        if (a.dx) {
            group_sum2<LANES>(mean_u, mean_uh, scratch);
            mean_u = a.centred ? mean_u * inv : 0.0f;
            mean_uh *= inv;
            X* dx = reinterpret_cast<X*>(a.dx) + row * a.width;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                float out[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) out[i] = r * (u[j][i] - mean_u - h[j][i] * mean_uh);
                const int64_t c = (lane + j * LANES) * VEC;
                if (c < a.width) store8(dx, c, a.width, out);
            }
        }
    }
    if (!a.partial) return;
    const int parts = a.with_bias ? 2 : 1;
    float* out = a.partial + static_cast<int64_t>(blockIdx.x) * parts * a.width;
    for (int part = 0; part < parts; ++part) {
        if constexpr (GROUPS > 1) {   // the groups' sums one after the other: a fixed order
            for (int n = 0; n < GROUPS; ++n) {
                __syncthreads();
                if (group == n) {
#pragma unroll
                    for (int j = 0; j < NV; ++j)
#pragma unroll
                        for (int i = 0; i < VEC; ++i) {
                            const int c = (lane + j * LANES) * VEC + i;
                            const float mine = part ? db[j][i] : dw[j][i];
                            joined[c] = n ? joined[c] + mine : mine;
                        }
                }
            }
            __syncthreads();
            for (int64_t c = threadIdx.x; c < a.width; c += BLOCK) out[part * a.width + c] = joined[c];
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int64_t c = (lane + j * LANES) * VEC;
                if (c < a.width) store8(out + part * a.width, c, a.width, part ? db[j] : dw[j]);
            }
        }
    }
}

// Rows wider than the registers: a workgroup takes one row for dx and adds its row into its partial sums in memory, which it alone
// reads and writes.
template <class X, class G>
__global__ __launch_bounds__(WIDE_THREADS) void norm_backward_long_kernel(const BackwardArgs a) {
    __shared__ float scratch[16];
    const float inv = 1.0f / static_cast<float>(a.width);
    float* dw = a.partial ? a.partial + static_cast<int64_t>(blockIdx.x) * (a.with_bias ? 2 : 1) * a.width : nullptr;
    float* db = a.partial && a.with_bias ? dw + a.width : nullptr;
    bool begun = false;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const X* x = reinterpret_cast<const X*>(a.x) + row * a.ld;
        const G* g = reinterpret_cast<const G*>(a.g) + row * a.width;
        const float mu = a.stats[2 * row], r = a.stats[2 * row + 1];
        float mean_u = 0.0f, mean_uh = 0.0f, h[VEC], u[VEC], w[VEC];
        for (int64_t c = threadIdx.x * VEC; c < a.width; c += WIDE_THREADS * VEC) {
            load8(h, x, c, a.width);
            load8(u, g, c, a.width);
#pragma unroll
            for (int i = 0; i < VEC; ++i) w[i] = 1.0f;
            if (a.weight) load8_as(w, a.weight, a.w_dtype, c, a.width);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                h[i] = (h[i] - mu) * r;
                mean_u = fmaf(u[i], w[i], mean_u);
                mean_uh = fmaf(u[i] * w[i], h[i], mean_uh);
                if (c + i < a.width) {
                    if (dw) dw[c + i] = (begun ? dw[c + i] : 0.0f) + u[i] * h[i];
                    if (db) db[c + i] = (begun ? db[c + i] : 0.0f) + u[i];
                }
            }
        }
        begun = true;
        if (!a.dx) continue;
        group_sum2<WIDE_THREADS>(mean_u, mean_uh, scratch);
        mean_u = a.centred ? mean_u * inv : 0.0f;
        mean_uh *= inv;
        X* dx = reinterpret_cast<X*>(a.dx) + row * a.width;
        for (int64_t c = threadIdx.x * VEC; c < a.width; c += WIDE_THREADS * VEC) {
            load8(h, x, c, a.width);
            load8(u, g, c, a.width);
#pragma unroll
            for (int i = 0; i < VEC; ++i) w[i] = 1.0f;
            if (a.weight) load8_as(w, a.weight, a.w_dtype, c, a.width);
#pragma unroll
            for (int i = 0; i < VEC; ++i) h[i] = r * (u[i] * w[i] - mean_u - (h[i] - mu) * r * mean_uh);
            store8(dx, c, a.width, h);
        }
    }
}

// dw[c] = sum over the workgroups' partial rows: 64 columns x 16 strands of rows per workgroup, the strands joined in order.
constexpr int STRANDS = 16;
__global__ __launch_bounds__(64 * STRANDS) void norm_reduce_kernel(const float* partial, int64_t count, int64_t width, int parts, void* dw, void* db,
                                                                   int dtype) {
    __shared__ float sums[STRANDS][64];
    const int lane = threadIdx.x & 63, strand = threadIdx.x >> 6, part = blockIdx.y;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 64 + lane;
    float s = 0.0f;
    if (c < width)
        for (int64_t n = strand; n < count; n += 8 * STRANDS) {   // eight loads in flight
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = n + i * STRANDS < count ? partial[((n + i * STRANDS) * parts + part) * width + c] : 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) s += v[i];
        }
    sums[strand][lane] = s;
    __syncthreads();
    if (strand != 0 || c >= width) return;
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < STRANDS; ++i) s += sums[i][lane];
    void* out = part ? db : dw;
    if (out == nullptr) return;
    if (dtype == KF_F32) reinterpret_cast<float*>(out)[c] = s;
    else if (dtype == KF_BF16) reinterpret_cast<__bf16*>(out)[c] = static_cast<__bf16>(s);
    else reinterpret_cast<_Float16*>(out)[c] = static_cast<_Float16>(s);
}

// ---- host -----------------------------------------------------------------------------------------------------------------
// workgroups of a launch: enough to fill 256 compute units several times, each with several rows, so that the weights (and the
// partial sums of a backward pass) are read (written) once per many rows
int64_t forward_groups(int64_t rows, int64_t width) { return std::min<int64_t>(width <= WAVE_MAX ? cdiv(rows, 4) : rows, 2048); }
int64_t backward_groups(int64_t rows, int64_t width) { return std::min<int64_t>(width <= WAVE_MAX ? cdiv(rows, 4) : rows, width <= WAVE_MAX ? 1024 : 512); }

template <class X, class Y>
int forward_as(const ForwardArgs& a, hipStream_t stream) {
    const unsigned grid = static_cast<unsigned>(forward_groups(a.rows, a.width));
    if (a.width <= 64 * VEC) norm_forward_kernel<X, Y, 64, 1><<<grid, THREADS, 0, stream>>>(a);
    else if (a.width <= 64 * VEC * 2) norm_forward_kernel<X, Y, 64, 2><<<grid, THREADS, 0, stream>>>(a);
    else if (a.width <= WAVE_MAX) norm_forward_kernel<X, Y, 64, 4><<<grid, THREADS, 0, stream>>>(a);
    else if (a.width <= WIDE_THREADS * VEC) norm_forward_kernel<X, Y, WIDE_THREADS, 1><<<grid, WIDE_THREADS, 0, stream>>>(a);
    else if (a.width <= WIDE_THREADS * VEC * 2) norm_forward_kernel<X, Y, WIDE_THREADS, 2><<<grid, WIDE_THREADS, 0, stream>>>(a);
    else if (a.width <= WIDE_MAX) norm_forward_kernel<X, Y, WIDE_THREADS, 4><<<grid, WIDE_THREADS, 0, stream>>>(a);
    else norm_forward_long_kernel<X, Y><<<grid, WIDE_THREADS, 0, stream>>>(a);
    return launch_status();
}

template <class X, class G>
int backward_as(const BackwardArgs& a, hipStream_t stream) {
    const unsigned grid = static_cast<unsigned>(backward_groups(a.rows, a.width));
    if (a.width <= 64 * VEC) norm_backward_kernel<X, G, 64, 1><<<grid, THREADS, 0, stream>>>(a);
    else if (a.width <= 64 * VEC * 2) norm_backward_kernel<X, G, 64, 2><<<grid, THREADS, 0, stream>>>(a);
    else if (a.width <= WAVE_MAX) norm_backward_kernel<X, G, 64, 4><<<grid, THREADS, 0, stream>>>(a);
    else if (a.width <= WIDE_THREADS * VEC) norm_backward_kernel<X, G, WIDE_THREADS, 1><<<grid, WIDE_THREADS, 0, stream>>>(a);
    else if (a.width <= WIDE_THREADS * VEC * 2) norm_backward_kernel<X, G, WIDE_THREADS, 2><<<grid, WIDE_THREADS, 0, stream>>>(a);
    else if (a.width <= WIDE_MAX) norm_backward_kernel<X, G, WIDE_THREADS, 4><<<grid, WIDE_THREADS, 0, stream>>>(a);
    else norm_backward_long_kernel<X, G><<<grid, WIDE_THREADS, 0, stream>>>(a);
    return launch_status();
}

bool norm_type(int d) { return d == KF_F32 || d == KF_BF16 || d == KF_F16; }

// f(first, second) with the two element types as values
template <class F>
int with_types(int first, int second, F f) {
    auto inner = [&](auto x) {
        switch (second) {
            case KF_F32: return f(x, float());
            case KF_BF16: return f(x, __bf16());
            default: return f(x, static_cast<_Float16>(0));
        }
    };
    switch (first) {
        case KF_F32: return inner(float());
        case KF_BF16: return inner(__bf16());
        default: return inner(static_cast<_Float16>(0));
    }
}

}  // namespace

extern "C" {

int kf_norm_forward(void* y, int y_dtype, float* stats, const void* x, int x_dtype, int64_t rows, int64_t width, int64_t row_stride, const void* weight,
                    const void* bias, int w_dtype, int centred, float eps, void* stream) {
    if (!norm_type(x_dtype) || !norm_type(y_dtype) || ((weight || bias) && !norm_type(w_dtype))) return KF_ERR_UNSUPPORTED_DTYPE;
    if (y == nullptr || x == nullptr || rows <= 0 || width <= 0 || row_stride < 0 || !(eps >= 0.0f) || !isfinite(eps)) return KF_ERR_INVALID_ARGUMENT;
    const ForwardArgs a = {y, stats, x, weight, bias, rows, width, row_stride, w_dtype, centred != 0, eps};
    return with_types(x_dtype, y_dtype, [&](auto s, auto d) { return forward_as<decltype(s), decltype(d)>(a, reinterpret_cast<hipStream_t>(stream)); });
}

int64_t kf_norm_backward_workspace_bytes(int64_t rows, int64_t width) {
    return rows > 0 && width > 0 ? backward_groups(rows, width) * 2 * width * 4 : 0;
}

int kf_norm_backward(void* dx, void* dweight, void* dbias, const void* grad, int grad_dtype, const void* x, int x_dtype, const float* stats, int64_t rows,
                     int64_t width, int64_t row_stride, const void* weight, int w_dtype, int centred, void* workspace, int64_t workspace_bytes,
                     void* stream) {
    if (!norm_type(x_dtype) || !norm_type(grad_dtype) || ((weight || dweight || dbias) && !norm_type(w_dtype))) return KF_ERR_UNSUPPORTED_DTYPE;
    if (grad == nullptr || x == nullptr || stats == nullptr || rows <= 0 || width <= 0 || row_stride < 0) return KF_ERR_INVALID_ARGUMENT;
    const bool sums = dweight != nullptr || dbias != nullptr;
    if (dx == nullptr && !sums) return KF_OK;
    if (sums && (workspace == nullptr || workspace_bytes < kf_norm_backward_workspace_bytes(rows, width))) return KF_ERR_WORKSPACE_TOO_SMALL;
    const int with_bias = dbias != nullptr;
    const BackwardArgs a = {dx, sums ? reinterpret_cast<float*>(workspace) : nullptr, stats, grad, x, weight, rows, width, row_stride, w_dtype,
                            centred != 0, with_bias};
    const hipStream_t on = reinterpret_cast<hipStream_t>(stream);
    if (int s = with_types(x_dtype, grad_dtype, [&](auto t, auto g) { return backward_as<decltype(t), decltype(g)>(a, on); })) return s;
    if (!sums) return KF_OK;
    if (cdiv(width, 64) > 0x7fffffff) return KF_ERR_INVALID_ARGUMENT;
    norm_reduce_kernel<<<dim3(static_cast<unsigned>(cdiv(width, 64)), with_bias + 1), 64 * STRANDS, 0, on>>>(
        a.partial, backward_groups(rows, width), width, with_bias + 1, dweight, dbias, w_dtype);
    return launch_status();
}

}  // extern "C"
