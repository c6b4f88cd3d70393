// Root-mean-square norm over the channels of a row, with the residual's addition in front and, if asked, 8-bit output
// with scales behind; and its gradient.
//
//   h = round(x + residual),  rstd = (mean(h^2) + eps)^-1/2,  y = h * rstd * weight
//   u = dy * weight:  dx = rstd * (u - h * rstd^2 * mean(u * h)) + dresidual,  dweight = sum over rows of dy * h * rstd
//
// Both are bound by memory: the forward pass reads x and the residual once and writes h and y (or its codes) once, the
// backward pass reads dy, h and what reaches h past the norm once and writes dx once.  A row therefore stays in
// registers between its reduction and its stores: tpr threads hold NV vectors of VEC elements each.  The norm is taken
// of the sum as it is stored, rounded to the tensor's type, because that is what the backward pass and the next layer
// read.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "pxe_types.cuh"

namespace pxe {
namespace {

constexpr int kMaxChannels = 262144;
constexpr int kMaxGroup = 128;                             // channels that share a scale, but for whole rows
// Rows of the weight gradient's workspace, one for each block: about 9.7 MB of them, but at least 148 and at most 1184 (one
// and eight for each SM).
inline int max_partials(int channels) { return std::max(148, std::min(1184, 2424832 / channels)); }

struct NormParams {
    const void* x;
    const void* residual;
    const void* weight;
    void* h;
    void* y;
    uint8_t* q;
    float* scale;
    float* rstd;
    long long xs, rs, hs, ys, qs, rows;
    int channels, weight_f32, group, groups, group_shift;  // group = 1 << group_shift, or 0 for the row
    float eps, inv_channels;
};

struct NormBackParams {
    const void* dy;
    const void* h;
    const void* dres;
    const void* weight;
    const float* rstd;
    void* dx;
    float* partial;
    long long dys, hs, rs, dxs, rows;
    int channels, weight_f32;
    float inv_channels;
};

// Sum (or NaN-keeping maximum) over the blockDim.x threads of one row (a power of two up to a warp, or whole warps); `red`
// holds a float for each warp of the row.  Every thread of the block calls it.  One barrier: calls alternate between two
// places for `red`, so that a place is written again only after the barrier of the call in between, which all its readers
// have passed.
template <bool MAX>
__device__ __forceinline__ float row_reduce(float v, float* red)
{
    if (blockDim.x < 32) {
        for (int o = blockDim.x >> 1; o > 0; o >>= 1) {
            const float t = __shfl_xor_sync(0xffffffffu, v, o);
            v = MAX ? max_nan(v, t) : v + t;
        }
        return v;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float t = __shfl_xor_sync(0xffffffffu, v, o);
        v = MAX ? max_nan(v, t) : v + t;
    }
    if (blockDim.x == 32) return v;
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = (threadIdx.x & 31) < warps ? red[threadIdx.x & 31] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float u = __shfl_xor_sync(0xffffffffu, t, o);
        t = MAX ? max_nan(t, u) : t + u;
    }
    return t;
}

template <typename T, int VEC>
__device__ __forceinline__ void load_weight(const void* weight, int weight_f32, int col, float (&w)[VEC])
{
    if (weight == nullptr) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) w[j] = 1.0f;
    } else if (weight_f32) {
        const float* p = static_cast<const float*>(weight) + col;
        if constexpr (VEC == 8) {
            float a[4], b[4];
            unpack<float, 4>(gldv<uint4>(p), a);
            unpack<float, 4>(gldv<uint4>(p + 4), b);
#pragma unroll
            for (int j = 0; j < 4; ++j) { w[j] = a[j]; w[4 + j] = b[j]; }
        } else {
            unpack<float, VEC>(gldv<Raw<float, VEC>>(p), w);
        }
    } else {
        unpack<T, VEC>(gldv<Raw<T, VEC>>(static_cast<const T*>(weight) + col), w);
    }
}

// A thread's elements two an instruction, where there are two.
template <int VEC>
__device__ __forceinline__ float sum_squares(const float (&v)[VEC], float sum)
{
    if constexpr (VEC >= 2) {
        unsigned long long s2 = pair(sum, 0.0f);
#pragma unroll
        for (int j = 0; j < VEC; j += 2) {
            const unsigned long long p = pair(v[j], v[j + 1]);
            s2 = fma2(p, p, s2);
        }
        float a, b;
        unpair(s2, a, b);
        return a + b;
    } else {
        return fmaf(v[0], v[0], sum);
    }
}
template <int VEC>
__device__ __forceinline__ void scale_by(float (&v)[VEC], float rstd, const float (&w)[VEC])
{
    if constexpr (VEC >= 2) {
        const unsigned long long r2 = pair(rstd, rstd);
#pragma unroll
        for (int j = 0; j < VEC; j += 2) unpair(mul2(mul2(pair(v[j], v[j + 1]), r2), pair(w[j], w[j + 1])), v[j], v[j + 1]);
    } else {
        v[0] = v[0] * rstd * w[0];
    }
}
__device__ __forceinline__ float warp_largest(float v)
{
    float r;
    asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
template <int VEC>
__device__ __forceinline__ float largest_of(const float (&v)[VEC])
{
    float m = fabsf(v[0]);
#pragma unroll
    for (int j = 1; j < VEC; ++j) m = max_nan(m, fabsf(v[j]));
    return m;
}

// The first of a thread's NV vectors: a warp's vectors lie together, 32 to an access, so that one address serves them all.
template <int VEC, int NV>
__device__ __forceinline__ int first_column()
{
    return ((threadIdx.x & ~31u) * NV + (threadIdx.x & 31u)) * VEC;
}

// ---------------------------------------------------------------- forward, row in registers
// 16384 x 4096 bf16 with a residual: 82 us, the copy rate; to 8 bits with a scale for every 128 channels 74 us (0.98);
// 262144 x 128: 42 us (1.00).  Rows of an odd length go element by element and are bound by issue: 20000 x 1001 bf16 at
// 0.68 of the copy rate, to 8 bits 0.40.
// blockDim = (tpr, rows per block); short rows share a warp.  One row to a thread and no loop: what hides a row's loads is
// the SM's other blocks and those that follow (20000 x 1001 bf16: 38 us, against 71 with a loop over rows and the next row
// loaded ahead, which needs another row's registers and halves the blocks of an SM).
constexpr int kMaxRowsPerBlock = 8;                        // of more than a warp each

// EARLY: the weights are on their way before the row's sum is known, for launches that leave the SMs half empty (333 x 1023
// fp32: 2.6 us against 3.7); with many blocks the registers count for more (262144 x 128 bf16: 43.2 us against 41.4).
template <typename T, int VEC, int NV, bool Q, bool EARLY>
__global__ void __launch_bounds__(512, NV * VEC <= 16 ? 2 : 1)
rms_norm_kernel(const NormParams p)
{
    constexpr int SPAN = 32 * VEC;
    __shared__ float reds[kMaxRowsPerBlock][16], red_max[kMaxRowsPerBlock][16];
    extern __shared__ unsigned int group_max[];            // Q, groups that no set of lanes of one warp covers: [rpb][groups]
    const int slot = blockDim.x > 32 ? threadIdx.y : 0, C = p.channels, col0 = first_column<VEC, NV>();
    const long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y;
    const int mine = row < p.rows ? C - col0 : 0;          // vector i is there when i * SPAN < mine
    const T* const x = static_cast<const T*>(p.x) + row * p.xs + col0;
    const T* const r = static_cast<const T*>(p.residual) + row * p.rs + col0;
    Raw<T, VEC> xr[NV], rr[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (i * SPAN < mine) {
            xr[i] = gldv<Raw<T, VEC>>(x + i * SPAN);
            if (p.residual) rr[i] = gldv<Raw<T, VEC>>(r + i * SPAN);
        }
    }
    float w[EARLY ? NV : 1][VEC];
    if constexpr (EARLY) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (i * SPAN < mine) load_weight<T, VEC>(p.weight, p.weight_f32, col0 + i * SPAN, w[i]);
    }
    float v[NV][VEC];
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (i * SPAN < mine) {
            unpack<T, VEC>(xr[i], v[i]);
            if (p.residual) {
                float a[VEC];
                unpack<T, VEC>(rr[i], a);
#pragma unroll
                for (int j = 0; j < VEC; ++j) a[j] += v[i][j];
                const Raw<T, VEC> raw = pack<T, VEC>(a);
                gstv(static_cast<T*>(p.h) + row * p.hs + col0 + i * SPAN, raw);
                unpack<T, VEC>(raw, v[i]);
            }
            sum = sum_squares<VEC>(v[i], sum);
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[i][j] = 0.0f;
        }
    }
    sum = row_reduce<false>(sum, reds[slot]);
    const float rstd = rsqrtf(sum * p.inv_channels + p.eps);
    if (p.rstd && mine > 0 && threadIdx.x == 0) gst(p.rstd + row, rstd);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (i * SPAN < mine) {
            if constexpr (!EARLY) load_weight<T, VEC>(p.weight, p.weight_f32, col0 + i * SPAN, w[0]);
            scale_by<VEC>(v[i], rstd, w[EARLY ? i : 0]);
            if constexpr (!Q) gstv(static_cast<T*>(p.y) + row * p.ys + col0 + i * SPAN, pack<T, VEC>(v[i]));
        }
    }
    if constexpr (Q) {
        uint8_t* const q = p.q + row * p.qs + col0;
        auto store = [&](int i, float scale) {
            const float inv = e4m3_inverse(scale);
            float a[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) a[j] = v[i][j] * inv;
            gstv(q + i * SPAN, pack_e4m3<VEC>(a));
        };
        if (p.group == 0) {
            float largest = 0.0f;
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (i * SPAN < mine) largest = max_nan(largest, largest_of<VEC>(v[i]));
            const float scale = e4m3_scale(row_reduce<true>(largest, red_max[slot]));
            if (mine > 0 && threadIdx.x == 0) gst(p.scale + row, scale);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (i * SPAN < mine) store(i, scale);
        } else if (p.group <= 32 * VEC) {                  // a group is group / VEC neighbouring lanes of one warp
            const int lanes = p.group / VEC;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float m = i * SPAN < mine ? largest_of<VEC>(v[i]) : 0.0f;
                for (int o = lanes >> 1; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
                if (i * SPAN < mine) {
                    const float scale = e4m3_scale(m);
                    if ((threadIdx.x & (lanes - 1)) == 0) gst(p.scale + row * p.groups + ((col0 + i * SPAN) >> p.group_shift), scale);
                    store(i, scale);
                }
            }
        } else if constexpr (32 * VEC < kMaxGroup) {       // fp32 bits of |y| order as integers do, NaN above everything
            unsigned int* gm = group_max + threadIdx.y * p.groups;
            for (int g = threadIdx.x; g < p.groups; g += blockDim.x) gm[g] = 0u;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const float m = warp_largest(i * SPAN < mine ? largest_of<VEC>(v[i]) : 0.0f);      // (a warp lies within a group)
                if (i * SPAN < mine && (threadIdx.x & 31) == 0) atomicMax(gm + ((col0 + i * SPAN) >> p.group_shift), __float_as_uint(m));
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int col = col0 + i * SPAN;
                if (i * SPAN < mine) {
                    const float scale = e4m3_scale(__uint_as_float(gm[col >> p.group_shift]));
                    if ((col & (p.group - 1)) == 0) gst(p.scale + row * p.groups + (col >> p.group_shift), scale);
                    store(i, scale);
                }
            }
        }
    }
}

// ---------------------------------------------------------------- forward, any row length
// A block of 1024 threads per row; the row is read again (from L2 or from h) for its output.
template <typename T, int VEC, bool Q>
__global__ void __launch_bounds__(1024)
rms_norm_long_kernel(const NormParams p)
{
    __shared__ float red[32], red_max[32];
    extern __shared__ unsigned int group_max[];
    const int C = p.channels, step = blockDim.x * VEC, first = threadIdx.x * VEC;
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(p.x) + row * p.xs;
        const T* r = static_cast<const T*>(p.residual) + row * p.rs;
        T* h = static_cast<T*>(p.h) + row * p.hs;
        const T* again = p.residual ? h : x;
        float sum = 0.0f, v[VEC], w[VEC];
        for (int col = first; col < C; col += step) {
            unpack<T, VEC>(gldv<Raw<T, VEC>>(x + col), v);
            if (p.residual) {
                float a[VEC];
                unpack<T, VEC>(gldv<Raw<T, VEC>>(r + col), a);
#pragma unroll
                for (int j = 0; j < VEC; ++j) a[j] += v[j];
                const Raw<T, VEC> raw = pack<T, VEC>(a);
                gstv(h + col, raw);
                unpack<T, VEC>(raw, v);
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) sum = fmaf(v[j], v[j], sum);
        }
        __syncthreads();
        sum = row_reduce<false>(sum, red);
        const float rstd = rsqrtf(sum * p.inv_channels + p.eps);
        if (p.rstd && threadIdx.x == 0) gst(p.rstd + row, rstd);
        auto value = [&](int col) {
            unpack<T, VEC>(gldv<Raw<T, VEC>>(again + col), v);
            load_weight<T, VEC>(p.weight, p.weight_f32, col, w);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = v[j] * rstd * w[j];
        };
        if constexpr (!Q) {
            for (int col = first; col < C; col += step) {
                value(col);
                gstv(static_cast<T*>(p.y) + row * p.ys + col, pack<T, VEC>(v));
            }
        } else {
            __syncthreads();
            for (int g = threadIdx.x; g < p.groups; g += blockDim.x) group_max[g] = 0u;
            __syncthreads();
            float largest = 0.0f;
            for (int col = first; col < C; col += step) {
                value(col);
                const float m = largest_of<VEC>(v);
                if (p.group) atomicMax(group_max + (col >> p.group_shift), __float_as_uint(m));
                else largest = max_nan(largest, m);
            }
            if (!p.group) {
                largest = row_reduce<true>(largest, red_max);
                if (threadIdx.x == 0) group_max[0] = __float_as_uint(largest);
            }
            __syncthreads();
            for (int col = first; col < C; col += step) {
                value(col);
                const float scale = e4m3_scale(__uint_as_float(group_max[col >> p.group_shift]));
                if (col == (col >> p.group_shift) << p.group_shift) gst(p.scale + row * p.groups + (col >> p.group_shift), scale);
                const float inv = e4m3_inverse(scale);
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] *= inv;
                gstv(p.q + row * p.qs + col, pack_e4m3<VEC>(v));
            }
            __syncthreads();
        }
    }
}

// ---------------------------------------------------------------- backward, row in registers
// dx = rstd * u - h * (rstd * k) + dresidual with k = rstd^2 * mean(u * h), and the block's part of dweight in registers
// over all its rows.  Up to 8 elements a thread (HOLD) u and h stay in registers as floats, the weights with them, and the
// next row is loaded before this one is reduced; beyond that a row is held as it was loaded and converted twice.
// 262144 x 128 bf16: 52 us, 0.80 of the copy rate, bound by issue; 4096 x 16384: 110 us (0.75), where a block's one row is
// read, reduced and written in turn.
template <typename T, int VEC>
__device__ __forceinline__ void times(float (&a)[VEC], const float (&w)[VEC])
{
    if constexpr (VEC >= 2) {
#pragma unroll
        for (int j = 0; j < VEC; j += 2) unpair(mul2(pair(a[j], a[j + 1]), pair(w[j], w[j + 1])), a[j], a[j + 1]);
    } else {
        a[0] *= w[0];
    }
}
// acc += dy * h * rstd;  dy becomes u = dy * w;  returns dot + the sum of u * h
template <typename T, int VEC>
__device__ __forceinline__ float first_pass(float (&dy)[VEC], const float (&h)[VEC], const float (&w)[VEC], float rstd, float (&acc)[VEC], float dot)
{
    if constexpr (VEC >= 2) {
        const unsigned long long r2 = pair(rstd, rstd);
        unsigned long long d2 = pair(dot, 0.0f);
#pragma unroll
        for (int j = 0; j < VEC; j += 2) {
            const unsigned long long dy2 = pair(dy[j], dy[j + 1]), h2 = pair(h[j], h[j + 1]);
            unpair(fma2(dy2, mul2(h2, r2), pair(acc[j], acc[j + 1])), acc[j], acc[j + 1]);
            const unsigned long long u2 = mul2(dy2, pair(w[j], w[j + 1]));
            d2 = fma2(u2, h2, d2);
            unpair(u2, dy[j], dy[j + 1]);
        }
        float d0, d1;
        unpair(d2, d0, d1);
        return d0 + d1;
    } else {
        acc[0] = fmaf(dy[0], h[0] * rstd, acc[0]);
        dy[0] *= w[0];
        return fmaf(dy[0], h[0], dot);
    }
}
// u becomes u * rstd + (h * k + res)
template <int VEC>
__device__ __forceinline__ void second_pass(float (&u)[VEC], const float (&h)[VEC], const float (&res)[VEC], float rstd, float k)
{
    if constexpr (VEC >= 2) {
        const unsigned long long r2 = pair(rstd, rstd), k2 = pair(k, k);
#pragma unroll
        for (int j = 0; j < VEC; j += 2)
            unpair(fma2(pair(u[j], u[j + 1]), r2, fma2(pair(h[j], h[j + 1]), k2, pair(res[j], res[j + 1]))), u[j], u[j + 1]);
    } else {
        u[0] = fmaf(u[0], rstd, fmaf(h[0], k, res[0]));
    }
}

// A block's part of dweight to its row of the workspace; `shared`: a row of floats where the block has several rows, which
// are added one after the other, in a fixed order.
template <int VEC, int NV>
__device__ __forceinline__ void store_partial(const float (&acc)[NV][VEC], float* out, int C, int col0, float* shared)
{
    constexpr int SPAN = 32 * VEC;
    auto each = [&](auto&& f) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (col0 + i * SPAN + j < C) f(col0 + i * SPAN + j, acc[i][j]);
    };
    if (blockDim.y == 1) {
        if constexpr (VEC >= 4) {                          // (channels are a multiple of VEC)
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < VEC; j += 4)
                    if (col0 + i * SPAN < C) gstv(out + col0 + i * SPAN + j, make_float4(acc[i][j], acc[i][j + 1], acc[i][j + 2], acc[i][j + 3]));
        } else {
            each([&](int c, float v) { gst(out + c, v); });
        }
        return;
    }
    __syncthreads();
    for (int y = 0; y < (int)blockDim.y; ++y) {
        if ((int)threadIdx.y == y) each([&](int c, float v) { shared[c] = y == 0 ? v : shared[c] + v; });
        __syncthreads();
    }
    for (int c = threadIdx.y * blockDim.x + threadIdx.x; c < C; c += blockDim.x * blockDim.y) gst(out + c, shared[c]);
}

template <typename T, int VEC, int NV>
__global__ void __launch_bounds__(512, NV == 1 ? 2 : 1)    // (NV == 1: 262144 x 128 bf16 53 us against 78)
rms_norm_backward_kernel(const NormBackParams p)
{
    constexpr bool HOLD = NV * VEC <= 8;
    constexpr int SPAN = 32 * VEC;
    __shared__ float reds[2][kMaxRowsPerBlock][16];
    const int slot = blockDim.x > 32 ? threadIdx.y : 0;
    extern __shared__ float shared_dw[];                   // rows per block > 1: [channels]
    const int rpb = blockDim.y, C = p.channels, col0 = first_column<VEC, NV>();
    const T* const pdy = static_cast<const T*>(p.dy) + col0;
    const T* const ph = static_cast<const T*>(p.h) + col0;
    const T* const pres = p.dres ? static_cast<const T*>(p.dres) + col0 : nullptr;
    float acc[NV][VEC], w[HOLD ? NV : 1][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[i][j] = 0.0f;
    if constexpr (HOLD) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = col0 + i * SPAN;
            if (col < C) load_weight<T, VEC>(p.weight, p.weight_f32, col, w[i]);
        }
    }
    Raw<T, VEC> dyr[NV], hr[NV], resr[NV];
    float next_rstd = 0.0f;
    auto load = [&](long long row) {
        if (row >= p.rows) return;
        next_rstd = gld(p.rstd + row);
        const T* const dy = pdy + row * p.dys;
        const T* const h = ph + row * p.hs;
        const T* const res = pres + row * p.rs;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = col0 + i * SPAN;
            if (col < C) {
                dyr[i] = gldv<Raw<T, VEC>>(dy + i * SPAN);
                hr[i] = gldv<Raw<T, VEC>>(h + i * SPAN);
                if (pres) resr[i] = gldv<Raw<T, VEC>>(res + i * SPAN);
            }
        }
    };
    const long long step = (long long)gridDim.x * rpb;
    if (HOLD) load((long long)blockIdx.x * rpb + threadIdx.y);
    int turn = 0;
    for (long long row0 = (long long)blockIdx.x * rpb; row0 < p.rows; row0 += step, turn ^= 1) {
        const long long row = row0 + threadIdx.y;
        const bool active = row < p.rows;
        T* const dx = static_cast<T*>(p.dx) + row * p.dxs + col0;
        if (!HOLD) load(row);
        float u[HOLD ? NV : 1][VEC], h[HOLD ? NV : 1][VEC], res[HOLD ? NV : 1][VEC];
        auto unpack_residual = [&](int i) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) res[HOLD ? i : 0][j] = 0.0f;
            if (pres) unpack<T, VEC>(resr[i], res[HOLD ? i : 0]);
        };
        const float rstd = next_rstd;
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = col0 + i * SPAN, k = HOLD ? i : 0;
            if (active && col < C) {
                if constexpr (!HOLD) load_weight<T, VEC>(p.weight, p.weight_f32, col, w[0]);
                unpack<T, VEC>(dyr[i], u[k]);
                unpack<T, VEC>(hr[i], h[k]);
                if constexpr (HOLD) unpack_residual(i);
                dot = first_pass<T, VEC>(u[k], h[k], w[k], rstd, acc[i], dot);
            }
        }
        if (HOLD) load(row + step);
        dot = row_reduce<false>(dot, reds[turn][slot]);
        const float factor = -(dot * p.inv_channels * rstd * rstd * rstd);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = col0 + i * SPAN, k = HOLD ? i : 0;
            if (active && col < C) {
                if constexpr (!HOLD) {
                    load_weight<T, VEC>(p.weight, p.weight_f32, col, w[0]);
                    unpack<T, VEC>(dyr[i], u[0]);
                    unpack<T, VEC>(hr[i], h[0]);
                    unpack_residual(i);
                    times<T, VEC>(u[0], w[0]);
                }
                second_pass<VEC>(u[k], h[k], res[k], rstd, factor);
                gstv(dx + i * SPAN, pack<T, VEC>(u[k]));
            }
        }
    }
    if (p.partial == nullptr) return;
    store_partial<VEC, NV>(acc, p.partial + (long long)blockIdx.x * C, C, col0, shared_dw);
}

// Any row length: the row is read twice, the block's part of the weight gradient lives in its row of the workspace.
template <typename T, int VEC>
__global__ void __launch_bounds__(1024)
rms_norm_backward_long_kernel(const NormBackParams p)
{
    __shared__ float red[32];
    const int C = p.channels, step = blockDim.x * VEC, first = threadIdx.x * VEC;
    float* out = p.partial ? p.partial + (long long)blockIdx.x * C : nullptr;
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* dy = static_cast<const T*>(p.dy) + row * p.dys;
        const T* h = static_cast<const T*>(p.h) + row * p.hs;
        const float rstd = gld(p.rstd + row);
        float a[VEC], b[VEC], w[VEC], dot = 0.0f;
        for (int col = first; col < C; col += step) {
            unpack<T, VEC>(gldv<Raw<T, VEC>>(dy + col), a);
            unpack<T, VEC>(gldv<Raw<T, VEC>>(h + col), b);
            load_weight<T, VEC>(p.weight, p.weight_f32, col, w);
#pragma unroll
            for (int j = 0; j < VEC; ++j) dot = fmaf(a[j] * w[j], b[j], dot);
        }
        __syncthreads();
        dot = row_reduce<false>(dot, red);
        const float k = dot * p.inv_channels * rstd * rstd;
        for (int col = first; col < C; col += step) {
            unpack<T, VEC>(gldv<Raw<T, VEC>>(dy + col), a);
            unpack<T, VEC>(gldv<Raw<T, VEC>>(h + col), b);
            load_weight<T, VEC>(p.weight, p.weight_f32, col, w);
            if (out) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float t = a[j] * (b[j] * rstd);
                    gst(out + col + j, row == blockIdx.x ? t : gld(out + col + j) + t);
                }
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) a[j] = rstd * (a[j] * w[j] - b[j] * k);
            if (p.dres) {
                unpack<T, VEC>(gldv<Raw<T, VEC>>(static_cast<const T*>(p.dres) + row * p.rs + col), b);
#pragma unroll
                for (int j = 0; j < VEC; ++j) a[j] += b[j];
            }
            gstv(static_cast<T*>(p.dx) + row * p.dxs + col, pack<T, VEC>(a));
        }
    }
}

// ---------------------------------------------------------------- backward, many rows of whole vectors: a ring of rows in shared memory
// A block has to go over many rows (its part of dweight is in its registers), and the form above waits for one row while it
// works on another: too few bytes are on their way (a row's chain of load, barrier, reduction and store takes about 1.5 us,
// whatever it moves).  Here one thread keeps `stages` rows of every input coming in with bulk copies.  A row's barrier in
// its reduction says that all threads are done with the row before, whose place is then refilled.  Waits are bounded: where a
// copy does not complete, the block leaves NaN in that row of dx, in all its later ones and in its part of dweight, starts
// no further copy, and waits, bounded too, for those under way, which end in its shared memory.  16384 x 4096 bf16: 82 us,
// the copy rate, against 91 by the form above; 4096 x 8192: 46 against 74; 16384 x 1024: 27.4 against 27.9.  (Several short
// rows to a stage, filled by a warp, were slower than the form above: 44 against 28 us at 8192 x 2048.)
constexpr int kMaxStages = 8;
constexpr int kWaitLimit = 1 << 18;                        // tries of 4 us each: about a second

__device__ __forceinline__ uint32_t shared_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

struct Ring {
    unsigned char* data;                                   // [stages][stage_bytes]
    unsigned long long* full;                              // [stages]
    int stages, stage_bytes;
    __device__ __forceinline__ void init() const
    {
        if (threadIdx.x == 0) {
            for (int i = 0; i < stages; ++i) asm volatile("mbarrier.init.shared.b64 [%0], 1;" ::"r"(shared_address(full + i)) : "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        __syncthreads();
    }
    // One thread: a row of `bytes` bytes of each of n tensors into a stage.
    template <int N>
    __device__ __forceinline__ void fill(int stage, const void* const (&src)[N], int n, int bytes) const
    {
        const uint32_t bar = shared_address(full + stage);
        int expected = 0;
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (k < n && gcheck_range(src[k], bytes)) expected += bytes;
        asm volatile("mbarrier.arrive.expect_tx.shared.b64 _, [%0], %1;" ::"r"(bar), "r"(expected) : "memory");
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (k < n && gcheck_range(src[k], bytes))
                asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                                 shared_address(data + stage * stage_bytes + k * bytes)),
                             "l"(src[k]), "r"(bytes), "r"(bar)
                             : "memory");
    }
    __device__ __forceinline__ bool wait(int stage, int parity) const
    {
        const uint32_t bar = shared_address(full + stage);
        for (int i = 0; i < kWaitLimit; ++i) {
            uint32_t done;
            asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
                         : "=r"(done)
                         : "r"(bar), "r"(parity)
                         : "memory");
            if (done) return true;
        }
        return false;
    }
    template <typename V>
    static __device__ __forceinline__ V read(const unsigned char* p) { return *reinterpret_cast<const V*>(p); }
};

extern __shared__ __align__(128) unsigned char ring_shared[];

template <typename T>
__global__ void __launch_bounds__(1024, 1)                   // (an SM holds 1024 threads of any of its blocks: 64 registers each)
rms_norm_backward_ring_kernel(const NormBackParams p, int stages)
{
    constexpr int VEC = 16 / sizeof(T);                    // a thread holds one vector of the row
    __shared__ float reds[2][32];
    __shared__ unsigned long long full[kMaxStages];
    __shared__ int missing[2];                             // a thread's wait ran out (alternating as reds do)
    const int C = p.channels, col = threadIdx.x * VEC, bytes = C * (int)sizeof(T), inputs = p.dres ? 3 : 2;
    const bool there = col < C;
    const Ring ring{ring_shared, full, stages, bytes * inputs};
    if (threadIdx.x < 2) missing[threadIdx.x] = 0;
    ring.init();
    auto fill = [&](int stage, long long row) {
        const void* const src[3] = {static_cast<const T*>(p.dy) + row * p.dys, static_cast<const T*>(p.h) + row * p.hs,
                                    static_cast<const T*>(p.dres) + row * p.rs};
        ring.fill<3>(stage, src, inputs, bytes);
    };
    const long long step = gridDim.x;
    if (threadIdx.x == 0)
        for (int i = 0; i < stages; ++i)
            if (blockIdx.x + i * step < p.rows) fill(i, blockIdx.x + i * step);
    float acc[1][VEC], w[VEC], u[VEC], h[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[0][j] = u[j] = h[j] = 0.0f;
    if (there) load_weight<T, VEC>(p.weight, p.weight_f32, col, w);
    float next_rstd = gld(p.rstd + blockIdx.x);            // (there are at least two rows for each block)
    int stage = 0, parity = 0, turn = 0;
    long long row = blockIdx.x;
    for (; row < p.rows; row += step, turn ^= 1) {
        const float rstd = next_rstd;
        if (row + step < p.rows) next_rstd = gld(p.rstd + row + step);
        if (!ring.wait(stage, parity)) missing[turn] = 1;
        const unsigned char* const at = ring.data + stage * ring.stage_bytes + col * (int)sizeof(T);
        float dot = 0.0f;
        if (there) {
            unpack<T, VEC>(ring.read<Raw<T, VEC>>(at), u);
            unpack<T, VEC>(ring.read<Raw<T, VEC>>(at + bytes), h);
            dot = first_pass<T, VEC>(u, h, w, rstd, acc[0], dot);
        }
        dot = row_reduce<false>(dot, reds[turn]);
        if (missing[turn]) break;                          // the same for all: written before the barrier, or two rows later
        const int before = stage == 0 ? stages - 1 : stage - 1;
        if (threadIdx.x == 0 && row != blockIdx.x && row + (stages - 1) * step < p.rows) fill(before, row + (stages - 1) * step);
        if (there) {
            float res[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) res[j] = 0.0f;
            if (p.dres) unpack<T, VEC>(ring.read<Raw<T, VEC>>(at + 2 * bytes), res);
            second_pass<VEC>(u, h, res, rstd, -(dot * p.inv_channels * rstd * rstd * rstd));
            gstv(static_cast<T*>(p.dx) + row * p.dxs + col, pack<T, VEC>(u));
        }
        if (++stage == stages) { stage = 0; parity ^= 1; }
    }
    if (row < p.rows) {                                    // given up
        // under way: this row's copies and the next rows', as far as they were started (from the first row, one more)
        const int started = row == blockIdx.x ? stages : stages - 1;
        if (threadIdx.x == 0)
            for (int i = 0; i < started && row + i * step < p.rows; ++i) ring.wait((stage + i) % stages, parity ^ (stage + i >= stages));
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[0][j] = u[j] = __int_as_float(0x7fffffff);
        for (; there && row < p.rows; row += step) gstv(static_cast<T*>(p.dx) + row * p.dxs + col, pack<T, VEC>(u));
    }
    if (p.partial) store_partial<VEC, 1>(acc, p.partial + (long long)blockIdx.x * C, C, col, nullptr);
}

// dweight[c] = the sum of column c over the workspace's rows.  A block takes 32 columns, eight threads of four columns side
// by side (one 128-byte line of a row) and 128 rows at a time; then each warp's four row groups and the 32 warps are added
// in order.  Launched while the kernel that fills the workspace still runs; it waits for that one's end.  3.5 us of the 26
// that 8192 x 2048 bf16 takes, bound by the latency of the few loads that each thread has under way.
constexpr int kSumThreads = 1024;
__global__ void __launch_bounds__(kSumThreads)
rms_norm_dweight_kernel(const float* partial, int parts, int channels, float* dweight, int accumulate)
{
    __shared__ float part[32][33];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, c = blockIdx.x * 32 + (t & 7) * 4;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    cudaGridDependencySynchronize();
    if (channels % 4 == 0) {
        if (c < channels) {
#pragma unroll 5
            for (int r = t >> 3; r < parts; r += kSumThreads / 8) {
                float f[4];
                unpack<float, 4>(gldv<uint4>(partial + (long long)r * channels + c), f);
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[j] += f[j];
            }
        }
    } else {
        for (int r = t >> 3; r < parts; r += kSumThreads / 8)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c + j < channels) sum[j] += gld(partial + (long long)r * channels + c + j);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 8);
        sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 16);
        if (lane < 8) part[warp][lane * 4 + j] = sum[j];
    }
    __syncthreads();
    float total = part[lane][warp];                        // column `warp` of the block: a lane for each warp's sum
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    const int column = blockIdx.x * 32 + warp;
    if (lane == 0 && column < channels) gst(dweight + column, accumulate ? gld(dweight + column) + total : total);
}

// ---------------------------------------------------------------- host
// Widest access that a tensor's pointer and row stride allow (bytes, a power of two up to 16).
int widest(const void* p, long long stride_bytes)
{
    if (!p) return 16;
    const unsigned long long bits = reinterpret_cast<uintptr_t>(p) | (unsigned long long)stride_bytes | 16ull;
    return (int)(bits & (~bits + 1));
}

struct Layout {
    int vec;        // elements per access
    int nv;         // vectors per thread; 0: the row does not fit, the long form
    int tpr, rpb;
};

// Threads and registers for rows of `channels`.  What a row costs whatever its length (two trees of shuffles, a barrier)
// wants few threads with much each: rows that a warp holds with up to eight accesses or 32 bytes of a tensor a lane take a
// warp (or the power of two of its lanes that is enough); longer ones 128 threads with up to four vectors, then as many
// threads as they need, up to 512 (16384 x 4096 bf16: 82 us with four vectors, 91 with two).  With `few` rows (less than
// one for each SM), where nothing but a row's own time counts, one access up to 512 threads (64 x 4096 bf16: 2.2 us, 3.2
// by the rule for many); backward, where a thread holds three tensors and a sum for each element, 8 elements first.
Layout layout_for(int vec, int size, int channels, bool few, bool backward)
{
    Layout l{vec, 1, 32, 1};
    const int vecs = (channels + vec - 1) / vec, most = backward ? std::min(8, 8 / vec) : std::min(8, 32 / (vec * size));
    if (vecs <= 32) {
        l.tpr = 1;
        while (l.tpr < vecs) l.tpr *= 2;
        l.rpb = 256 / l.tpr;
        return l;
    }
    if (!few) {
        while (l.nv < most && l.nv * 32 < vecs) l.nv *= 2;
        if (l.nv * 32 >= vecs) {
            l.rpb = 8;
            return l;
        }
        while (!backward && l.nv < 4 && l.nv * 128 < vecs) l.nv *= 2;
    }
    while (l.nv * 512 < vecs) l.nv *= 2;
    if (l.nv > 8 || l.nv * vec * size > 64) {
        l.nv = 0;
        l.tpr = 1024;
        return l;
    }
    l.tpr = ((vecs + l.nv - 1) / l.nv + 31) / 32 * 32;
    l.rpb = l.tpr <= 128 ? std::min(kMaxRowsPerBlock, 256 / l.tpr) : 1;
    return l;
}

// The ring form takes rows of 2 to 16 KB in whole vectors (shorter ones would need more blocks than the workspace has rows),
// when there are enough of them to fill the card: a thread for each vector, 1024 threads to an SM, and the stages that seven
// eighths of the shared memory hold.  (Rows of 32 KB leave room for two stages: 121 us against 113 for the form above at
// 4096 x 16384 bf16.)
struct RingLayout {
    int threads, blocks_per_sm, stages;
    size_t shared;
};
bool ring_layout(int size, int channels, int inputs, long long rows, const DeviceInfo& di, RingLayout* l)
{
    const int bytes = channels * size;
    if (bytes < 2048 || bytes > 16384) return false;
    l->threads = (bytes / 16 + 31) / 32 * 32;
    l->blocks_per_sm = 1024 / l->threads;
    if (rows < 2LL * di.sm_count * l->blocks_per_sm) return false;
    l->stages = (int)std::min<long long>(kMaxStages, (long long)di.max_smem_optin * 7 / 8 / l->blocks_per_sm / (bytes * inputs));
    l->shared = (size_t)l->stages * bytes * inputs;
    return l->stages >= 2;
}

// Allows a kernel its dynamic shared memory, once for each device.
template <typename K>
int allow_shared(K kernel, int device, int bytes, std::atomic<unsigned long long>& done)
{
    if (done.load(std::memory_order_relaxed) >> device & 1) return PXE_OK;
    PXE_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done.fetch_or(1ull << device, std::memory_order_relaxed);
    return PXE_OK;
}

template <typename T>
int launch_backward_ring(cudaStream_t s, const NormBackParams& p, const RingLayout& l, const DeviceInfo& di, int device)
{
    static std::atomic<unsigned long long> done{0};
    { const int rc = allow_shared(rms_norm_backward_ring_kernel<T>, device, di.max_smem_optin - 4096, done); if (rc != PXE_OK) return rc; }
    rms_norm_backward_ring_kernel<T><<<(unsigned)(di.sm_count * l.blocks_per_sm), l.threads, l.shared, s>>>(p, l.stages);
    PXE_LAUNCH_OK("rms_norm_backward_ring_kernel");
    return PXE_OK;
}

template <typename T, int VEC, bool Q>
int launch_norm(cudaStream_t s, const NormParams& p, const Layout& l, const DeviceInfo& di)
{
    const size_t group_bytes = Q ? (size_t)std::max(1, p.groups) * 4 : 0;
    if (l.nv == 0) {
        const unsigned grid = (unsigned)std::min<long long>(p.rows, 2LL * di.sm_count);
        rms_norm_long_kernel<T, VEC, Q><<<grid, 1024, group_bytes, s>>>(p);
        PXE_LAUNCH_OK("rms_norm_long_kernel");
        return PXE_OK;
    }
    const long long blocks = (p.rows + l.rpb - 1) / l.rpb;
    PXE_REQUIRE(blocks <= 0x7fffffffLL, "rms_norm: too many rows");
    const size_t smem = Q && p.group > 32 * VEC ? group_bytes * l.rpb : 0;
    const dim3 block(l.tpr, l.rpb);
    auto launch = [&](auto nv) {
        constexpr int NV = decltype(nv)::value;
        if (NV * VEC <= 16 && blocks <= 4LL * di.sm_count) rms_norm_kernel<T, VEC, NV, Q, NV * VEC <= 16><<<(unsigned)blocks, block, smem, s>>>(p);
        else rms_norm_kernel<T, VEC, NV, Q, false><<<(unsigned)blocks, block, smem, s>>>(p);
    };
    switch (l.nv) {
    case 1: launch(std::integral_constant<int, 1>{}); break;
    case 2: launch(std::integral_constant<int, 2>{}); break;
    case 4: launch(std::integral_constant<int, 4>{}); break;
    default:
        if constexpr (VEC <= 2) launch(std::integral_constant<int, 8>{});
        break;
    }
    PXE_LAUNCH_OK("rms_norm_kernel");
    return PXE_OK;
}

template <typename T, int VEC>
int launch_backward(cudaStream_t s, const NormBackParams& p, const Layout& l, unsigned grid)
{
    if (l.nv == 0) {
        rms_norm_backward_long_kernel<T, VEC><<<grid, 1024, 0, s>>>(p);
        PXE_LAUNCH_OK("rms_norm_backward_long_kernel");
        return PXE_OK;
    }
    const size_t smem = l.rpb > 1 && p.partial ? (size_t)p.channels * 4 : 0;
    const dim3 block(l.tpr, l.rpb);
    switch (l.nv) {
    case 1: rms_norm_backward_kernel<T, VEC, 1><<<grid, block, smem, s>>>(p); break;
    case 2: rms_norm_backward_kernel<T, VEC, 2><<<grid, block, smem, s>>>(p); break;
    case 4: rms_norm_backward_kernel<T, VEC, 4><<<grid, block, smem, s>>>(p); break;
    default:
        if constexpr (VEC <= 2) rms_norm_backward_kernel<T, VEC, 8><<<grid, block, smem, s>>>(p);
        break;
    }
    PXE_LAUNCH_OK("rms_norm_backward_kernel");
    return PXE_OK;
}

template <typename T>
int launch_backward_16(cudaStream_t s, const NormBackParams& p, const Layout& l, unsigned grid, int vec)
{
    if (vec == 8) return launch_backward<T, 8>(s, p, l, grid);
    return vec == 2 ? launch_backward<T, 2>(s, p, l, grid) : launch_backward<T, 1>(s, p, l, grid);
}

// Elements per access: the whole 16 bytes, 4, or one element, whichever alignment, strides and channels allow.
int vec_for(int access, int channels, int size)
{
    int vec = 16 / size;
    while (vec > 1 && (vec * size > access || channels % vec != 0)) vec /= 2;
    return vec == 4 && size == 2 ? 2 : vec == 2 && size == 4 ? 1 : vec;
}

}  // namespace
}  // namespace pxe

using namespace pxe;

extern "C" int pxe_rms_norm(pxe_stream_t stream, const pxe_rms_norm_desc* dp)
{
    PXE_REQUIRE(dp != nullptr, "rms_norm: null descriptor");
    const pxe_rms_norm_desc& d = *dp;
    PXE_REQUIRE(valid_dtype(d.type), "rms_norm: unknown type %d", d.type);
    PXE_REQUIRE(d.weight_type == PXE_F32 || d.weight_type == d.type, "rms_norm: weight_type %d is neither fp32 nor the tensor's", d.weight_type);
    PXE_REQUIRE(d.rows >= 0 && d.channels > 0, "rms_norm: shape [%lld, %d]", d.rows, d.channels);
    PXE_REQUIRE((d.y != nullptr) != (d.q != nullptr), "rms_norm: exactly one of y and q is the destination");
    PXE_REQUIRE(d.eps >= 0.0f, "rms_norm: eps is negative or NaN");
    PXE_REQUIRE(!d.q || d.group == 0 || d.group == 32 || d.group == 64 || d.group == kMaxGroup, "rms_norm: group %d is not 0, 32, 64 or 128", d.group);
    if (d.channels > kMaxChannels) return set_error(PXE_ERR_UNSUPPORTED, "rms_norm: %d channels, at most %d", d.channels, kMaxChannels);
    if (d.rows == 0) return PXE_OK;
    PXE_REQUIRE(d.x != nullptr, "rms_norm: x is null");
    PXE_REQUIRE((d.residual != nullptr) == (d.h != nullptr), "rms_norm: a residual and h come together");
    PXE_REQUIRE(!d.q || d.scale != nullptr, "rms_norm: q without scale");
    const int size = dtype_bytes(d.type), C = d.channels;
    NormParams p{};
    p.x = d.x; p.residual = d.residual; p.weight = d.weight; p.h = d.h; p.y = d.y; p.q = static_cast<uint8_t*>(d.q);
    p.scale = d.scale; p.rstd = d.rstd;
    p.rows = d.rows; p.channels = C; p.weight_f32 = d.weight_type == PXE_F32;
    p.group = d.q && d.group < C ? d.group : 0;            // one group is the row
    p.groups = p.group ? (C + p.group - 1) / p.group : 1;
    p.group_shift = p.group == 32 ? 5 : p.group == 64 ? 6 : p.group == 128 ? 7 : 30;
    p.eps = d.eps; p.inv_channels = 1.0f / (float)C;
    const struct { const char* name; const void* ptr; long long given; long long* stride; int bytes; } tensors[] = {
        {"x", d.x, d.x_row_stride, &p.xs, size}, {"residual", d.residual, d.residual_row_stride, &p.rs, size},
        {"h", d.h, d.h_row_stride, &p.hs, size}, {"y", d.y, d.y_row_stride, &p.ys, size}, {"q", d.q, d.q_row_stride, &p.qs, 1}};
    RowSpan span[5];
    int access = 16;
    for (int i = 0; i < 5; ++i) {
        const auto& t = tensors[i];
        *t.stride = t.given ? t.given : C;
        span[i] = {t.ptr, d.rows, *t.stride * t.bytes, (long long)C * t.bytes};
        if (!t.ptr) continue;
        PXE_REQUIRE(*t.stride >= C, "rms_norm: %s_row_stride %lld is less than %d channels", t.name, t.given, C);
        const int w = widest(t.ptr, *t.stride * t.bytes);
        PXE_REQUIRE(w >= t.bytes, "rms_norm: %s is not aligned to its elements", t.name);
        access = std::min(access, w * size / t.bytes);                     // one byte of q for an element of the others
    }
    PXE_REQUIRE(!rows_conflict(span[2], span[0]) && !rows_conflict(span[2], span[1]), "rms_norm: h partially overlaps a source");
    PXE_REQUIRE(!rows_conflict(span[3], span[0]) && !rows_conflict(span[3], span[1]), "rms_norm: y partially overlaps a source");
    PXE_REQUIRE(!(d.y && d.y == d.h) && !rows_conflict(span[3], span[2]), "rms_norm: y overlaps h");
    for (int i = 0; i < 3; ++i)
        PXE_REQUIRE(!(d.q && d.q == tensors[i].ptr) && !rows_conflict(span[4], span[i]), "rms_norm: q overlaps %s", tensors[i].name);
    const int wsize = p.weight_f32 ? 4 : size;
    PXE_REQUIRE(!d.weight || widest(d.weight, 0) >= wsize, "rms_norm: weight is not aligned to its elements");
    int vec = vec_for(access, C, size);
    if (d.weight && widest(d.weight, 0) < std::min(16, vec * wsize)) vec = 1;
    const RowSpan stats{d.rstd, 1, 0, d.rows * 4}, scales{d.q ? d.scale : nullptr, 1, 0, d.rows * p.groups * 4}, weights{d.weight, 1, 0, (long long)C * wsize};
    PXE_REQUIRE(((uintptr_t)d.rstd | (uintptr_t)scales.p) % 4 == 0, "rms_norm: rstd or scale is not aligned to its elements");
    PXE_REQUIRE(!rows_conflict(stats, scales) && !(scales.p && scales.p == d.rstd) && !rows_conflict(stats, weights) && !rows_conflict(scales, weights) &&
                !(d.weight && (d.weight == d.rstd || d.weight == scales.p)), "rms_norm: rstd, scale and weight overlap");
    for (int i = 2; i < 5; ++i)
        PXE_REQUIRE(!rows_conflict(span[i], weights) && !(d.weight && tensors[i].ptr == d.weight), "rms_norm: %s overlaps the weight", tensors[i].name);
    for (int i = 0; i < 5; ++i)
        PXE_REQUIRE(!(tensors[i].ptr && (tensors[i].ptr == d.rstd || (d.q && tensors[i].ptr == d.scale))) && !rows_conflict(span[i], stats) &&
                    !(d.q && rows_conflict(span[i], scales)), "rms_norm: rstd or scale overlaps %s", tensors[i].name);
    DeviceInfo di;
    { const int rc = device_info(&di); if (rc != PXE_OK) return rc; }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const Layout l = layout_for(vec, size, C, d.rows < di.sm_count, false);
#define PXE_NORM_VEC(T, V) return d.q ? launch_norm<T, V, true>(s, p, l, di) : launch_norm<T, V, false>(s, p, l, di)
    if (d.type == PXE_F32) { if (vec == 4) PXE_NORM_VEC(float, 4); PXE_NORM_VEC(float, 1); }
    if (d.type == PXE_BF16) { if (vec == 8) PXE_NORM_VEC(bf16, 8); if (vec == 2) PXE_NORM_VEC(bf16, 2); PXE_NORM_VEC(bf16, 1); }
    if (vec == 8) PXE_NORM_VEC(f16, 8);
    if (vec == 2) PXE_NORM_VEC(f16, 2);
    PXE_NORM_VEC(f16, 1);
#undef PXE_NORM_VEC
}

extern "C" size_t pxe_rms_norm_backward_workspace_bytes(long long rows, int channels)
{
    if (rows <= 0 || channels <= 0) return 0;
    return (size_t)std::min<long long>(rows, max_partials(channels)) * channels * 4;
}

extern "C" int pxe_rms_norm_backward(pxe_stream_t stream, const pxe_rms_norm_backward_desc* dp)
{
    PXE_REQUIRE(dp != nullptr, "rms_norm_backward: null descriptor");
    const pxe_rms_norm_backward_desc& d = *dp;
    PXE_REQUIRE(valid_dtype(d.type), "rms_norm_backward: unknown type %d", d.type);
    PXE_REQUIRE(d.weight_type == PXE_F32 || d.weight_type == d.type, "rms_norm_backward: weight_type %d is neither fp32 nor the tensor's", d.weight_type);
    PXE_REQUIRE(d.rows >= 0 && d.channels > 0, "rms_norm_backward: shape [%lld, %d]", d.rows, d.channels);
    if (d.channels > kMaxChannels) return set_error(PXE_ERR_UNSUPPORTED, "rms_norm_backward: %d channels, at most %d", d.channels, kMaxChannels);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int size = dtype_bytes(d.type), C = d.channels;
    PXE_REQUIRE(!d.dweight || widest(d.dweight, 0) >= 4, "rms_norm_backward: dweight is not aligned to its elements");
    if (d.rows == 0) {
        if (d.dweight && !d.accumulate) PXE_CUDA_OK(cudaMemsetAsync(d.dweight, 0, (size_t)C * 4, s));
        return PXE_OK;
    }
    PXE_REQUIRE(d.dy && d.h && d.rstd && d.dx, "rms_norm_backward: null pointer");
    NormBackParams p{};
    p.dy = d.dy; p.h = d.h; p.dres = d.dresidual; p.weight = d.weight; p.rstd = d.rstd; p.dx = d.dx;
    p.rows = d.rows; p.channels = C; p.weight_f32 = d.weight_type == PXE_F32; p.inv_channels = 1.0f / (float)C;
    const struct { const char* name; const void* ptr; long long given; long long* stride; } tensors[] = {
        {"dy", d.dy, d.dy_row_stride, &p.dys}, {"h", d.h, d.h_row_stride, &p.hs},
        {"dresidual", d.dresidual, d.dresidual_row_stride, &p.rs}, {"dx", d.dx, d.dx_row_stride, &p.dxs}};
    RowSpan span[4];
    int access = 16;
    for (int i = 0; i < 4; ++i) {
        const auto& t = tensors[i];
        *t.stride = t.given ? t.given : C;
        span[i] = {t.ptr, d.rows, *t.stride * size, (long long)C * size};
        if (!t.ptr) continue;
        PXE_REQUIRE(*t.stride >= C, "rms_norm_backward: %s_row_stride %lld is less than %d channels", t.name, t.given, C);
        const int w = widest(t.ptr, *t.stride * size);
        PXE_REQUIRE(w >= size, "rms_norm_backward: %s is not aligned to its elements", t.name);
        access = std::min(access, w);
    }
    for (int i = 0; i < 3; ++i) PXE_REQUIRE(!rows_conflict(span[3], span[i]), "rms_norm_backward: dx partially overlaps %s", tensors[i].name);
    const int wsize = p.weight_f32 ? 4 : size;
    PXE_REQUIRE(!d.weight || widest(d.weight, 0) >= wsize, "rms_norm_backward: weight is not aligned to its elements");
    PXE_REQUIRE((uintptr_t)d.rstd % 4 == 0, "rms_norm_backward: rstd is not aligned to its elements");
    const RowSpan rstd{d.rstd, 1, 0, d.rows * 4}, weights{d.weight, 1, 0, (long long)C * wsize};
    PXE_REQUIRE(!rows_conflict(span[3], rstd) && !rows_conflict(span[3], weights) && d.dx != (const void*)d.rstd && d.dx != d.weight,
                "rms_norm_backward: dx overlaps rstd or the weight");
    const size_t need = d.dweight ? pxe_rms_norm_backward_workspace_bytes(d.rows, C) : 0;
    if (d.dweight) {
        PXE_REQUIRE(d.workspace && aligned16(d.workspace), "rms_norm_backward: dweight needs a 16-byte aligned workspace");
        if (d.workspace_bytes < need) return set_error(PXE_ERR_WORKSPACE, "rms_norm_backward: workspace of %zu bytes, %zu needed", d.workspace_bytes, need);
        const RowSpan ws{d.workspace, 1, 0, (long long)need}, dw{d.dweight, 1, 0, (long long)C * 4};
        for (int i = 0; i < 4; ++i)
            PXE_REQUIRE(!rows_conflict(ws, span[i]) && !rows_conflict(dw, span[i]) && d.workspace != tensors[i].ptr && d.dweight != tensors[i].ptr,
                        "rms_norm_backward: the workspace or dweight overlaps %s", tensors[i].name);
        PXE_REQUIRE(!rows_conflict(ws, dw) && d.workspace != (void*)d.dweight, "rms_norm_backward: the workspace overlaps dweight");
        PXE_REQUIRE(!rows_conflict(ws, rstd) && !rows_conflict(dw, rstd) && !rows_conflict(ws, weights) && !rows_conflict(dw, weights) &&
                    (const void*)d.dweight != d.weight && d.dweight != d.rstd, "rms_norm_backward: the workspace or dweight overlaps rstd or the weight");
    }
    p.partial = d.dweight ? static_cast<float*>(d.workspace) : nullptr;
    int vec = vec_for(access, C, size);
    if (d.weight && widest(d.weight, 0) < std::min(16, vec * wsize)) vec = 1;
    DeviceInfo di;
    { const int rc = device_info(&di); if (rc != PXE_OK) return rc; }
    int rc;
    unsigned grid;
    RingLayout rl;
    if (vec * size == 16 && ring_layout(size, C, d.dresidual ? 3 : 2, d.rows, di, &rl) && di.sm_count * rl.blocks_per_sm <= max_partials(C)) {
        int device = 0;
        PXE_CUDA_OK(cudaGetDevice(&device));
        grid = (unsigned)(di.sm_count * rl.blocks_per_sm);
        rc = d.type == PXE_F32 ? launch_backward_ring<float>(s, p, rl, di, device) : d.type == PXE_BF16 ? launch_backward_ring<bf16>(s, p, rl, di, device)
                                                                                                        : launch_backward_ring<f16>(s, p, rl, di, device);
    } else {
        const Layout l = layout_for(vec, size, C, false, true);
        const long long blocks = (d.rows + l.rpb - 1) / l.rpb;
        grid = (unsigned)std::min<long long>(std::min<long long>(blocks, max_partials(C)), (long long)di.sm_count * std::max(1, 1024 / (l.tpr * l.rpb)));
        if (d.type == PXE_F32) rc = vec == 4 ? launch_backward<float, 4>(s, p, l, grid) : launch_backward<float, 1>(s, p, l, grid);
        else rc = d.type == PXE_BF16 ? launch_backward_16<bf16>(s, p, l, grid, vec) : launch_backward_16<f16>(s, p, l, grid, vec);
    }
    if (rc != PXE_OK || !d.dweight) return rc;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((C + 31) / 32);
    cfg.blockDim = dim3(kSumThreads);
    cfg.stream = s;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    PXE_CUDA_OK(cudaLaunchKernelEx(&cfg, rms_norm_dweight_kernel, (const float*)p.partial, (int)grid, C, d.dweight, d.accumulate));
    return PXE_OK;
}
