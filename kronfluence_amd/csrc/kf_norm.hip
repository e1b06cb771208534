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
//
// Measured (a copy reaches 5.2 TB/s): 131072 x 768 bf16 -> fp32 forward 105 us (5.8 TB/s), backward 138 + 6 (5.8 TB/s); 16384 x 768 fp32
// forward 18 us, backward 27 + 6; RMS norm of 8192 x 4096 bf16 forward 25 us (5.4 TB/s), backward 41 + 4 (5.0 TB/s).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "../../include/kronfluence_hip.h"

namespace {

constexpr int THREADS = 256, WIDE_THREADS = 512;
// Columns a wave / a workgroup of WIDE_THREADS holds in registers (32 per lane).  One wave against eight: 16384 x 1100 fp32 forward 26
// and 38 us, backward 53 and 47; 8192 x 2048 bf16 16 and 21, 31 and 32.
constexpr int WAVE_MAX = 2048, WIDE_MAX = 16384;

// Columns per chunk: 16 bytes of the wider of the two types a kernel streams, so that every wave access to it is 1 KB without gaps
// (with 8 fp32 columns per lane a store instruction wrote every second 16 bytes: 131072 x 768 bf16 -> fp32 166 us).
template <class A, class B>
constexpr int vec_of() { return 16 / static_cast<int>(sizeof(A) > sizeof(B) ? sizeof(A) : sizeof(B)); }

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int launch_status() { return hipGetLastError() == hipSuccess ? KF_OK : KF_ERR_LAUNCH_FAILED; }

// VEC consecutive elements at any element-aligned address (rows of odd widths start anywhere).
template <class T, int VEC>
struct __attribute__((packed, aligned(sizeof(T)))) Chunk { T v[VEC]; };

template <int VEC, class T>
__device__ __forceinline__ Chunk<T, VEC> load_chunk(const T* p, int64_t column, int64_t width) {
    Chunk<T, VEC> c;
    if (column + VEC <= width) {
        c = *reinterpret_cast<const Chunk<T, VEC>*>(p + column);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) c.v[i] = column + i < width ? p[column + i] : static_cast<T>(0.0f);
    }
    return c;
}
template <int VEC, class T>
__device__ __forceinline__ void widen(float (&x)[VEC], const Chunk<T, VEC>& c) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[i] = static_cast<float>(c.v[i]);
}
template <int VEC, class T>
__device__ __forceinline__ void load(float (&x)[VEC], const T* p, int64_t column, int64_t width) { widen(x, load_chunk<VEC>(p, column, width)); }

// PAST: past the caches, for results that the kernel does not read again (131072 x 768 bf16 -> fp32: forward 152 us, 138 with it; backward
// 157 and 138; 16384 x 768 fp32: forward 21 and 18; what reads the result next is no slower: 2048 to 131072 rows, a product or a sum)
template <bool PAST, int VEC, class T>
__device__ __forceinline__ void store(T* p, int64_t column, int64_t width, const float (&x)[VEC]) {
    if (column + VEC <= width) {
        typedef T Vector __attribute__((ext_vector_type(VEC), aligned(sizeof(T))));
        Vector v;
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = static_cast<T>(x[i]);
        if constexpr (PAST) __builtin_nontemporal_store(v, reinterpret_cast<Vector*>(p + column));
        else *reinterpret_cast<Vector*>(p + column) = v;
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (column + i < width) p[column + i] = static_cast<T>(x[i]);
    }
}

// elements of a vector whose type is known at run time only (weight, bias: read once per workgroup)
template <int VEC>
__device__ __forceinline__ void load_as(float (&x)[VEC], const void* p, int dtype, int64_t column, int64_t width) {
    if (dtype == KF_F32) load(x, reinterpret_cast<const float*>(p), column, width);
    else if (dtype == KF_BF16) load(x, reinterpret_cast<const __bf16*>(p), column, width);
    else load(x, reinterpret_cast<const _Float16*>(p), column, width);
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
    constexpr int BLOCK = LANES > 64 ? LANES : THREADS, GROUPS = BLOCK / LANES, VEC = vec_of<X, Y>();
    __shared__ float scratch[16];
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    const float inv = 1.0f / static_cast<float>(a.width);
    float w[NV][VEC], b[NV][VEC];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int64_t c = (lane + j * LANES) * VEC;
#pragma unroll
        for (int i = 0; i < VEC; ++i) { w[j][i] = 1.0f; b[j][i] = 0.0f; }
        if (a.weight) load_as(w[j], a.weight, a.w_dtype, c, a.width);
        if (a.bias) load_as(b[j], a.bias, a.w_dtype, c, a.width);
    }
    const int64_t step = static_cast<int64_t>(gridDim.x) * GROUPS;
    int64_t row = static_cast<int64_t>(blockIdx.x) * GROUPS + group;
    Chunk<X, VEC> next[NV];   // the next row is on its way while this one is worked on
    auto fetch = [&](int64_t at) {
        const X* x = reinterpret_cast<const X*>(a.x) + at * a.ld;
#pragma unroll
        for (int j = 0; j < NV; ++j) next[j] = load_chunk<VEC>(x, (lane + j * LANES) * VEC, a.width);
    };
    if (row < a.rows) fetch(row);
    for (; row < a.rows; row += step) {
        float v[NV][VEC];
#pragma unroll
        for (int j = 0; j < NV; ++j) widen(v[j], next[j]);
        if (row + step < a.rows) fetch(row + step);
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
            if (c < a.width) store<true>(y, c, a.width, out);
        }
        if (a.stats && lane == 0) { a.stats[2 * row] = mu; a.stats[2 * row + 1] = r; }
    }
}

// Rows wider than the registers: the row is read three times (from memory once, then from the cache).
template <class X, class Y>
__global__ __launch_bounds__(WIDE_THREADS) void norm_forward_long_kernel(const ForwardArgs a) {
    constexpr int VEC = vec_of<X, Y>();
    __shared__ float scratch[16];
    const float inv = 1.0f / static_cast<float>(a.width);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const X* x = reinterpret_cast<const X*>(a.x) + row * a.ld;
        float mu = 0.0f, ss = 0.0f, v[VEC], w[VEC], b[VEC];
        if (a.centred) {
            for (int64_t c = threadIdx.x * VEC; c < a.width; c += WIDE_THREADS * VEC) {
                load(v, x, c, a.width);
#pragma unroll
                for (int i = 0; i < VEC; ++i) mu += v[i];
            }
            mu = group_sum<WIDE_THREADS>(mu, scratch) * inv;
        }
        for (int64_t c = threadIdx.x * VEC; c < a.width; c += WIDE_THREADS * VEC) {
            load(v, x, c, a.width);
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (c + i < a.width) ss = fmaf(v[i] - mu, v[i] - mu, ss);
        }
        const float r = 1.0f / sqrtf(group_sum<WIDE_THREADS>(ss, scratch) * inv + a.eps);
        Y* y = reinterpret_cast<Y*>(a.y) + row * a.width;
        for (int64_t c = threadIdx.x * VEC; c < a.width; c += WIDE_THREADS * VEC) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) { w[i] = 1.0f; b[i] = 0.0f; }
            if (a.weight) load_as(w, a.weight, a.w_dtype, c, a.width);
            if (a.bias) load_as(b, a.bias, a.w_dtype, c, a.width);
            load(v, x, c, a.width);
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[i] = fmaf((v[i] - mu) * r, w[i], b[i]);
            store<true>(y, c, a.width, v);
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
    constexpr int VEC = vec_of<X, G>(), BLOCK = LANES > 64 ? LANES : THREADS, GROUPS = BLOCK / LANES, COLUMNS = LANES * NV * VEC;
    __shared__ float scratch[16];
    __shared__ float joined[GROUPS > 1 ? COLUMNS : 1];
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    const float inv = 1.0f / static_cast<float>(a.width);
    float w[NV][VEC], dw[NV][VEC], db[NV][VEC];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) { w[j][i] = 1.0f; dw[j][i] = 0.0f; db[j][i] = 0.0f; }
        if (a.weight) load_as(w[j], a.weight, a.w_dtype, (lane + j * LANES) * VEC, a.width);
    }
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * GROUPS + group; row < a.rows; row += static_cast<int64_t>(gridDim.x) * GROUPS) {
        const X* x = reinterpret_cast<const X*>(a.x) + row * a.ld;
        const G* g = reinterpret_cast<const G*>(a.g) + row * a.width;
        const float mu = a.stats[2 * row], r = a.stats[2 * row + 1];
        float h[NV][VEC], u[NV][VEC], mean_u = 0.0f, mean_uh = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t c = (lane + j * LANES) * VEC;
            load(h[j], x, c, a.width);
            load(u[j], g, c, a.width);
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
                if (c < a.width) store<true>(dx, c, a.width, out);
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
                if (c < a.width) store<false>(out + part * a.width, c, a.width, part ? db[j] : dw[j]);
            }
        }
    }
}

// Rows wider than the registers: a workgroup takes one row for dx and adds its row into its partial sums in memory, which it alone
// reads and writes.
template <class X, class G>
__global__ __launch_bounds__(WIDE_THREADS) void norm_backward_long_kernel(const BackwardArgs a) {
    constexpr int VEC = vec_of<X, G>();
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
            load(h, x, c, a.width);
            load(u, g, c, a.width);
#pragma unroll
            for (int i = 0; i < VEC; ++i) w[i] = 1.0f;
            if (a.weight) load_as(w, a.weight, a.w_dtype, c, a.width);
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
            load(h, x, c, a.width);
            load(u, g, c, a.width);
#pragma unroll
            for (int i = 0; i < VEC; ++i) w[i] = 1.0f;
            if (a.weight) load_as(w, a.weight, a.w_dtype, c, a.width);
#pragma unroll
            for (int i = 0; i < VEC; ++i) h[i] = r * (u[i] * w[i] - mean_u - (h[i] - mu) * r * mean_uh);
            store<true>(dx, c, a.width, h);
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
// Workgroups of a launch: as many as the card holds at once, each with several rows, so that the weights (and the partial sums of a
// backward pass) are read (written) once per many rows and no second round is left half full (131072 x 768 bf16 -> fp32, 1536 at once:
// forward 105 us, 143 with 2048; backward, 1024 at once: 140, 205 with 512).  A backward pass takes at most MAX_PARTIALS, which the
// workspace has room for.
constexpr int64_t CUS = 256, MAX_PARTIALS = 1024;
template <auto KERNEL>
int64_t resident(int threads) {
    static const int64_t all = [threads] {
        int blocks = 0;
        return hipOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, KERNEL, threads, 0) == hipSuccess && blocks > 0 ? blocks * CUS : MAX_PARTIALS;
    }();
    return all;
}
int64_t row_groups(int64_t rows, int64_t width) { return width <= WAVE_MAX ? cdiv(rows, 4) : rows; }
int64_t most_partials(int64_t rows, int64_t width) { return std::min(row_groups(rows, width), MAX_PARTIALS); }

// f(LANES, NV) with the smallest group that holds a row of `width` columns in registers; LANES 0: none does
template <int VEC, class F>
void with_group(int64_t width, F f) {
    using std::integral_constant;
    const int64_t wave = cdiv(width, 64 * VEC), wide = cdiv(width, WIDE_THREADS * VEC);
    constexpr integral_constant<int, 64> one;
    constexpr integral_constant<int, WIDE_THREADS> eight;
    if (width > WIDE_MAX) return f(integral_constant<int, 0>(), integral_constant<int, 0>());
    if (width > WAVE_MAX) {
        if (wide == 1) return f(eight, integral_constant<int, 1>());
        if (wide == 2) return f(eight, integral_constant<int, 2>());
        if (wide <= 4) return f(eight, integral_constant<int, 4>());
        if constexpr (VEC < 8) return f(eight, integral_constant<int, 8>());
    }
    if (wave == 1) return f(one, integral_constant<int, 1>());
    if (wave == 2) return f(one, integral_constant<int, 2>());
    if constexpr (VEC < 8) {
        if (wave == 3) return f(one, integral_constant<int, 3>());
        if (wave > 4) return f(one, integral_constant<int, 8>());
    }
    f(one, integral_constant<int, 4>());
}

template <class X, class Y, int LANES, int NV>
constexpr auto forward_kernel() {
    if constexpr (LANES == 0) return &norm_forward_long_kernel<X, Y>;
    else return &norm_forward_kernel<X, Y, LANES, NV>;
}
template <class X, class G, int LANES, int NV>
constexpr auto backward_kernel() {
    if constexpr (LANES == 0) return &norm_backward_long_kernel<X, G>;
    else return &norm_backward_kernel<X, G, LANES, NV>;
}

template <class X, class Y>
int forward_as(const ForwardArgs& a, hipStream_t stream) {
    with_group<vec_of<X, Y>()>(a.width, [&](auto lanes, auto nv) {
        constexpr int threads = lanes == 64 ? THREADS : WIDE_THREADS;
        constexpr auto kernel = forward_kernel<X, Y, lanes, nv>();
        kernel<<<static_cast<unsigned>(std::min(row_groups(a.rows, a.width), resident<kernel>(threads))), threads, 0, stream>>>(a);
    });
    return launch_status();
}

// `groups`: the partial rows it writes
template <class X, class G>
int backward_as(const BackwardArgs& a, hipStream_t stream, int64_t& groups) {
    with_group<vec_of<X, G>()>(a.width, [&](auto lanes, auto nv) {
        constexpr int threads = lanes == 64 ? THREADS : WIDE_THREADS;
        constexpr auto kernel = backward_kernel<X, G, lanes, nv>();
        groups = std::min(most_partials(a.rows, a.width), resident<kernel>(threads));
        kernel<<<static_cast<unsigned>(groups), threads, 0, stream>>>(a);
    });
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
    return rows > 0 && width > 0 ? most_partials(rows, width) * 2 * width * 4 : 0;
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
    int64_t groups = 0;
    if (int s = with_types(x_dtype, grad_dtype, [&](auto t, auto g) { return backward_as<decltype(t), decltype(g)>(a, on, groups); })) return s;
    if (!sums) return KF_OK;
    if (cdiv(width, 64) > 0x7fffffff) return KF_ERR_INVALID_ARGUMENT;
    norm_reduce_kernel<<<dim3(static_cast<unsigned>(cdiv(width, 64)), with_bias + 1), 64 * STRANDS, 0, on>>>(
        a.partial, groups, width, with_bias + 1, dweight, dbias, w_dtype);
    return launch_status();
}

}  // extern "C"
