// An AdamW step over many tensors in one launch, with states in 32 or 8 bits.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,  p -= rate ((m / c1) / (sqrt(v / c2) + eps) + decay p)
//
// Bound by memory: every element's parameter, gradient and moments are read once and all but the gradient written once
// (28 bytes in fp32, 16 with states in 8 bits).  The tensors' addresses travel as the kernel's parameters (72 bytes
// each, 400 to a launch), so a call needs no table in device memory, no copy and no workspace, and a captured call keeps
// its own.  A block of 256 threads takes 2048 elements of one tensor, which it finds by bisection over the first block of
// each.  A warp takes 256 elements, eight to a lane: that is also the block of elements that shares a scale in 8 bits, so
// the new scale is one reduction over the warp and nothing is read twice.  There is no loop: what hides a warp's loads is
// the other warps of the SM and the blocks that follow.
//
// In 8 bits m is held as an e4m3 code times its block's scale, and v as the code of its root: the update needs the root,
// and its codes then reach 2^-18 of the block's largest value (2^-36 in v).  A v above zero keeps the smallest code
// instead of rounding to zero, which would leave a later step to divide by eps alone.  Codes are 6 to 12 % apart, and a step
// moves the root of v by 0.05 % (beta2 = 0.999): rounded to nearest, all of that is lost and the moments stand still.
// With a seed they are rounded up or down at random, each as likely as it is near, so that on average nothing is lost.
#include <algorithm>
#include <exception>
#include <type_traits>
#include <vector>

#include "pxe_types.cuh"

namespace pxe {
namespace {

constexpr int kUnit = PXE_ADAMW_BLOCK;                     // elements a warp takes at a time
constexpr int kThreads = 256;
constexpr int kElements = kThreads / 32 * kUnit;           // of a block

struct Entry {
    void* p;
    const void* g;
    void* m;
    void* v;
    float* ms;
    float* vs;
    float* w;
    long long n;
    int first_block;
    int vector;                                            // every pointer allows whole accesses
};

template <int MAX>
struct AdamwParams {
    float rate, b1, b2, omb1, omb2, eps, decay, grad_scale, inv_c1, inv_c2, log_b1, log_b2;
    const float* rate_device;
    const long long* t_device;
    const float* grad_scale_device;
    const float* skip_device;
    unsigned long long seed;
    long long t;
    int count, blocks, before;                             // tensors of this launch, their blocks, tensors of earlier launches
    Entry e[MAX];
};

// The hardware's root and reciprocal (one unit in the last place; subnormal arguments kept, unlike the .ftz forms): an
// update is off by a few units of 2^-23 of itself, far below the parameter's own rounding.  The decay is part of the update
// (as a factor 1 - rate * decay of p it would move in steps of 2^-24: 1.3 % too much at 1e-6, none at all below 2^-25).
__device__ __forceinline__ float root(float x)
{
    float y;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float reciprocal(float x)
{
    float y;
    asm("rcp.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

struct Step {
    float b1, b2, omb1, omb2, eps, shrink, grad_scale, step, inv_root_c2;         // shrink = -rate * decay, step = rate / c1
    // the new moments and parameter of one element, and the second moment's root
    __device__ __forceinline__ float operator()(float& p, float g, float& m, float& v) const
    {
        g *= grad_scale;
        m = fmaf(omb1, g, b1 * m);
        v = fmaf(omb2 * g, g, b2 * v);
        const float r = root(v);
        p += fmaf(shrink, p, -step * m * reciprocal(fmaf(r, inv_root_c2, eps)));
        return r;
    }
};

// A 32-bit integer hash: C. Wellons, "Prospecting for hash functions" (2018), the variant with two multiplications.
__device__ __forceinline__ uint32_t mix(uint32_t x)
{
    x ^= x >> 16;
    x *= 0x7feb352du;
    x ^= x >> 15;
    x *= 0x846ca68bu;
    return x ^ x >> 16;
}
__device__ __forceinline__ uint32_t mix(uint32_t x, unsigned long long next) { return mix(mix(x ^ (uint32_t)next) ^ (uint32_t)(next >> 32)); }

// a in [0, 448) to the e4m3 value below or above it by 16 random bits: they are added under the three bits of the mantissa
// that a code has (among the smallest codes, 2^-9 apart, after 2^-6 is added, where floats have those bits at 2^-9), and
// what lies under the three is cut off.  Too likely by 2^-17 at most.  Anything else as it is, for the conversion to round.
__device__ __forceinline__ float round_at_random(float a, uint32_t bits16)
{
    const float base = a < 0.015625f ? 0.015625f : 0.0f;
    const float q = __uint_as_float((__float_as_uint(a + base) + (bits16 << 4)) & 0xfff00000u) - base;
    return a < kE4m3Max ? fminf(q, kE4m3Max) : a;
}

__device__ __forceinline__ float warp_max(float v)
{
    float r;
    asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

// Eight elements of a lane as they lie in memory: COUNT accesses of N of them, STRIDE apart.
template <typename T, int N>
struct Raw8 {
    static constexpr int COUNT = 8 / N, STRIDE = 32 * N, PER = N * sizeof(T) > 16 ? 16 / (int)sizeof(T) : N, PIECES = N / PER;
    Raw<T, PER> raw[COUNT][PIECES];
    __device__ __forceinline__ void load(const T* p, long long left)              // the first `left` elements of the unit are there
    {
#pragma unroll
        for (int k = 0; k < COUNT; ++k)
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                raw[k][i] = Raw<T, PER>{};
                if (k * STRIDE < left) raw[k][i] = gldv<Raw<T, PER>>(p + k * STRIDE + i * PER);
            }
    }
    __device__ __forceinline__ void get(int k, float (&f)[N]) const
    {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            float part[PER];
            unpack<T, PER>(raw[k][i], part);
#pragma unroll
            for (int j = 0; j < PER; ++j) f[i * PER + j] = part[j];
        }
    }
};
template <typename T, int N>
__device__ __forceinline__ void store(T* p, const float (&f)[N])
{
    constexpr int PER = N * sizeof(T) > 16 ? 16 / (int)sizeof(T) : N;
#pragma unroll
    for (int i = 0; i < N / PER; ++i) {
        float part[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) part[j] = f[i * PER + j];
        gstv(p + i * PER, pack<T, PER>(part));
    }
}

// One unit of 256 elements of a warp: all its loads, then the work on them.  RANDOM: 8-bit codes are rounded at random, by a
// hash of `key` (of seed, step, tensor and unit) and the element's place in the unit.
template <typename P, typename G, bool SMALL, bool RANDOM, bool MASTER, int N>
struct Unit {
    using S = std::conditional_t<SMALL, uint8_t, float>;
    using W = std::conditional_t<MASTER, float, P>;
    static constexpr int COUNT = 8 / N, STRIDE = 32 * N;
    Raw8<W, N> w;
    Raw8<G, N> g;
    Raw8<S, N> m, v;
    float ms, vs;
    long long at, left;                                    // this lane's first element; how many of the unit's there are from it

    __device__ __forceinline__ void load(const Entry& e, long long first, int lane)
    {
        at = first + lane * N;
        left = N == 1 ? e.n - at : 256;
        if constexpr (MASTER) w.load(e.w + at, left);
        else w.load(static_cast<const P*>(e.p) + at, left);
        g.load(static_cast<const G*>(e.g) + at, left);
        m.load(static_cast<const S*>(e.m) + at, left);
        v.load(static_cast<const S*>(e.v) + at, left);
        if constexpr (SMALL) { ms = gld(e.ms + first / kUnit); vs = gld(e.vs + first / kUnit); }
    }
    __device__ __forceinline__ void work(const Entry& e, long long first, int lane, const Step& step, uint32_t key)
    {
        float m1[COUNT][N], v1[COUNT][N], m_max = 0.0f, v_max = 0.0f;
#pragma unroll
        for (int k = 0; k < COUNT; ++k) {
            float p[N], grad[N];
            w.get(k, p);
            g.get(k, grad);
            if constexpr (SMALL) {
                unpack_e4m3<N>(m.raw[k][0], m1[k]);
                unpack_e4m3<N>(v.raw[k][0], v1[k]);
#pragma unroll
                for (int j = 0; j < N; ++j) { m1[k][j] *= ms; v1[k][j] *= vs; v1[k][j] *= v1[k][j]; }
            } else {
                m.get(k, m1[k]);
                v.get(k, v1[k]);
            }
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float r = step(p[j], grad[j], m1[k][j], v1[k][j]);
                if constexpr (SMALL) v1[k][j] = r;
            }
            if (k * STRIDE < left) {
                if constexpr (MASTER) store<float, N>(e.w + at + k * STRIDE, p);
                store<P, N>(static_cast<P*>(e.p) + at + k * STRIDE, p);
                if constexpr (SMALL) {
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        m_max = max_nan(m_max, fabsf(m1[k][j]));
                        v_max = max_nan(v_max, v1[k][j]);
                    }
                } else {
                    store<float, N>(static_cast<float*>(e.m) + at + k * STRIDE, m1[k]);
                    store<float, N>(static_cast<float*>(e.v) + at + k * STRIDE, v1[k]);
                }
            }
        }
        if constexpr (SMALL) {
            const float m_scale = e4m3_scale(warp_max(m_max)), v_scale = e4m3_scale(warp_max(v_max));
            const float mi = e4m3_inverse(m_scale), vi = e4m3_inverse(v_scale);
            constexpr float kSmallest = 0.001953125f;      // 2^-9
            if (lane == 0) { gst(e.ms + first / kUnit, m_scale); gst(e.vs + first / kUnit, v_scale); }
#pragma unroll
            for (int k = 0; k < COUNT; ++k) {
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    m1[k][j] *= mi;
                    float r = v1[k][j] * vi;
                    if constexpr (RANDOM) {
                        const uint32_t h = mix(key ^ (uint32_t)(lane * N + k * STRIDE + j));
                        m1[k][j] = copysignf(round_at_random(fabsf(m1[k][j]), h & 0xffffu), m1[k][j]);
                        r = round_at_random(r, h >> 16);
                    }
                    v1[k][j] = v1[k][j] > 0.0f ? max_nan(r, kSmallest) : v1[k][j];
                }
                if (k * STRIDE < left) {
                    gstv(static_cast<uint8_t*>(e.m) + at + k * STRIDE, pack_e4m3<N>(m1[k]));
                    gstv(static_cast<uint8_t*>(e.v) + at + k * STRIDE, pack_e4m3<N>(v1[k]));
                }
            }
        }
    }
};

template <typename P, typename G, bool SMALL, bool RANDOM, bool MASTER, int N>
__device__ __forceinline__ void one_unit(const Entry& e, long long first, int lane, const Step& step, uint32_t key)
{
    Unit<P, G, SMALL, RANDOM, MASTER, N> u;
    u.load(e, first, lane);
    u.work(e, first, lane, step, key);
}

// 64 M elements in 16 tensors: fp32 with states in 32 bits 272 us, 1.07 of the copy rate; fp32 with states in 8 bits 164 us
// (1.02); bf16 with a master copy and states in 8 bits 164 us (1.02), without the copy 130 us (0.80, 10 bytes an element and as
// many instructions).  With a seed 236, 219 and 212 us: bound by the instructions of the hash and the roundings.
// Blocks of an SM: four (64 registers a thread, nothing spilled), six for 16-bit parameters with states in 8 bits, whose
// lanes have half the bytes under way (64 M bf16 parameters: 122 against 134 us, with a master copy 164 against 167; fp32
// parameters with states in 8 bits 157 against 171 us at six).
template <typename P, typename G, bool SMALL, bool RANDOM, bool MASTER, int MAX>
__global__ void __launch_bounds__(kThreads, SMALL && sizeof(P) == 2 ? 6 : 4)
adamw_kernel(const __grid_constant__ AdamwParams<MAX> a)
{
    if (a.skip_device && gld(a.skip_device) != 0.0f) return;
    if (a.t_device && gld(a.t_device) < 1) return;         // 1 - b^0 = 0 would divide
    // chosen as values: a member of Step overwritten under a condition kept the parameter's value (nvcc 12.9)
    const float rate = a.rate_device ? gld(a.rate_device) : a.rate;
    const float grad_scale = a.grad_scale_device ? gld(a.grad_scale_device) : a.grad_scale;
    float inv_c1 = a.inv_c1, inv_c2 = a.inv_c2;
    if (a.t_device) {                                      // 1 - b^t without the cancellation of the difference
        const float t = (float)gld(a.t_device);
        inv_c1 = -1.0f / expm1f(t * a.log_b1);
        inv_c2 = -1.0f / expm1f(t * a.log_b2);
    }
    const Step step{a.b1, a.b2, a.omb1, a.omb2, a.eps, -rate * a.decay, grad_scale, rate * inv_c1, sqrtf(inv_c2)};
    constexpr int N = sizeof(P) == 4 ? 4 : 8;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int lo = 0, hi = a.count;                              // the last entry that begins at or before this block's elements
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.e[mid].first_block <= (int)blockIdx.x) lo = mid; else hi = mid;
    }
    const Entry& e = a.e[lo];
    const long long first = (long long)((int)blockIdx.x - e.first_block) * kElements + warp * kUnit;
    if (first >= e.n) return;
    uint32_t key = 0;
    if constexpr (RANDOM) {
        const long long t = a.t_device ? gld(a.t_device) : a.t;
        key = mix(mix(mix(mix(0u, a.seed), (unsigned long long)t), (unsigned long long)(a.before + lo)), (unsigned long long)(first / kUnit));
    }
    if (e.vector && first + kUnit <= e.n) one_unit<P, G, SMALL, RANDOM, MASTER, N>(e, first, lane, step, key);
    else one_unit<P, G, SMALL, RANDOM, MASTER, 1>(e, first, lane, step, key);
}

using Params = AdamwParams<PXE_ADAMW_TENSORS_PER_LAUNCH>;

template <typename P, typename G, bool SMALL, bool RANDOM, bool MASTER>
int launch(cudaStream_t s, const Params& a)
{
    adamw_kernel<P, G, SMALL, RANDOM, MASTER, PXE_ADAMW_TENSORS_PER_LAUNCH><<<(unsigned)a.blocks, kThreads, 0, s>>>(a);
    PXE_LAUNCH_OK("adamw_kernel");
    return PXE_OK;
}

template <typename P, typename G, bool MASTER>
int launch(cudaStream_t s, const Params& a, bool small)
{
    if (!small) return launch<P, G, false, false, MASTER>(s, a);
    return a.seed ? launch<P, G, true, true, MASTER>(s, a) : launch<P, G, true, false, MASTER>(s, a);
}

template <typename P, typename G>
int launch(cudaStream_t s, const Params& a, bool small, bool master)
{
    if constexpr (sizeof(P) == 2) { if (master) return launch<P, G, true>(s, a, small); }
    return launch<P, G, false>(s, a, small);
}

struct Range {
    uintptr_t lo, hi;
    bool written;
};

// True when a written range shares a byte with any other.
bool ranges_conflict(std::vector<Range>& r)
{
    bool ordered = true;
    for (size_t i = 1; i < r.size() && ordered; ++i) ordered = r[i - 1].hi <= r[i].lo;
    if (ordered) return false;
    std::sort(r.begin(), r.end(), [](const Range& a, const Range& b) { return a.lo < b.lo; });
    uintptr_t any = 0, written = 0;                        // the furthest ends so far
    for (const Range& x : r) {
        if (x.lo < written || (x.written && x.lo < any)) return true;
        any = std::max(any, x.hi);
        if (x.written) written = std::max(written, x.hi);
    }
    return false;
}

}  // namespace
}  // namespace pxe

using namespace pxe;

extern "C" int pxe_adamw_update(pxe_stream_t stream, const pxe_adamw_desc* dp)
{
    PXE_REQUIRE(dp != nullptr, "adamw_update: null descriptor");
    const pxe_adamw_desc& d = *dp;
    PXE_REQUIRE(d.count >= 0 && (d.count == 0 || d.tensors), "adamw_update: null or negative list of tensors");
    PXE_REQUIRE(valid_dtype(d.param_type) && valid_dtype(d.grad_type), "adamw_update: unknown type");
    if (d.param_type != PXE_F32 && d.grad_type != d.param_type && d.grad_type != PXE_F32)
        return set_error(PXE_ERR_UNSUPPORTED, "adamw_update: gradients of one 16-bit type for parameters of the other");
    PXE_REQUIRE(d.state_bits == 32 || d.state_bits == 8, "adamw_update: state_bits %d is neither 32 nor 8", d.state_bits);
    PXE_REQUIRE(d.seed == 0 || d.state_bits == 8, "adamw_update: a seed rounds states in 8 bits only");
    PXE_REQUIRE(d.beta1 >= 0.0f && d.beta1 < 1.0f && d.beta2 >= 0.0f && d.beta2 < 1.0f, "adamw_update: beta1 and beta2 lie in [0, 1)");
    PXE_REQUIRE(d.eps >= 0.0f, "adamw_update: eps is negative or NaN");
    PXE_REQUIRE(d.t_device || d.t >= 1, "adamw_update: step %lld (the first step is 1)", d.t);
    PXE_REQUIRE(((uintptr_t)d.rate_device | (uintptr_t)d.grad_scale_device | (uintptr_t)d.skip_device) % 4 == 0 && (uintptr_t)d.t_device % 8 == 0,
                "adamw_update: a device scalar is not aligned to its type");
    const bool small = d.state_bits == 8;
    const int psize = dtype_bytes(d.param_type), gsize = dtype_bytes(d.grad_type), ssize = small ? 1 : 4;
    bool master = false, first = true;
    try {
        std::vector<Range> ranges;
        for (int family = 0; family < 7; ++family) {       // a family at a time: flat buffers come out in order
            for (int i = 0; i < d.count; ++i) {
                const pxe_adamw_tensor& t = d.tensors[i];
                PXE_REQUIRE(t.n >= 0, "adamw_update: tensor %d has %lld elements", i, t.n);
                if (t.n == 0) continue;
                const long long blocks = (t.n + kUnit - 1) / kUnit;
                if (family == 0) {
                    PXE_REQUIRE(t.param && t.grad && t.m && t.v, "adamw_update: tensor %d has a null pointer", i);
                    PXE_REQUIRE(small == (t.m_scale != nullptr) && small == (t.v_scale != nullptr), "adamw_update: tensor %d: scales come with 8-bit state", i);
                    if (first) { master = t.master != nullptr; first = false; }
                    PXE_REQUIRE(master == (t.master != nullptr), "adamw_update: a master copy in all tensors or in none");
                    PXE_REQUIRE(!master || d.param_type != PXE_F32, "adamw_update: a master copy of fp32 parameters");
                    PXE_REQUIRE(t.n <= (1LL << 40), "adamw_update: tensor %d has %lld elements", i, t.n);
                    PXE_REQUIRE((uintptr_t)t.param % psize == 0 && (uintptr_t)t.grad % gsize == 0 && ((uintptr_t)t.m | (uintptr_t)t.v) % ssize == 0 &&
                                ((uintptr_t)t.m_scale | (uintptr_t)t.v_scale | (uintptr_t)t.master) % 4 == 0,
                                "adamw_update: tensor %d is not aligned to its elements", i);
                }
                const void* p[7] = {t.param, t.grad, t.m, t.v, t.m_scale, t.v_scale, t.master};
                const long long bytes[7] = {t.n * psize, t.n * gsize, t.n * ssize, t.n * ssize, blocks * 4, blocks * 4, t.n * 4};
                if (p[family]) ranges.push_back({(uintptr_t)p[family], (uintptr_t)p[family] + (uintptr_t)bytes[family], family != 1});
            }
        }
        const struct { uintptr_t lo, bytes; } scalars[4] = {{(uintptr_t)d.rate_device, 4}, {(uintptr_t)d.t_device, 8},
                                                         {(uintptr_t)d.grad_scale_device, 4}, {(uintptr_t)d.skip_device, 4}};
        for (const auto& x : scalars)
            for (const Range& r : ranges)
                PXE_REQUIRE(!x.lo || !r.written || x.lo >= r.hi || x.lo + x.bytes <= r.lo, "adamw_update: a device scalar lies inside what the step writes");
        PXE_REQUIRE(!ranges_conflict(ranges), "adamw_update: tensors overlap (one listed twice, or a state, master or gradient inside another)");
    } catch (const std::exception& e) {
        return set_error(PXE_ERR_CUDA, "adamw_update: %s", e.what());
    }
    if (first) return PXE_OK;                              // nothing to do
    Params a;
    a.rate = d.rate; a.b1 = d.beta1; a.b2 = d.beta2; a.omb1 = (float)(1.0 - (double)d.beta1); a.omb2 = (float)(1.0 - (double)d.beta2);
    a.eps = d.eps; a.decay = d.weight_decay; a.grad_scale = d.grad_scale;
    a.log_b1 = (float)std::log((double)d.beta1); a.log_b2 = (float)std::log((double)d.beta2);
    a.inv_c1 = d.t_device ? 0.0f : (float)(1.0 / (1.0 - std::pow((double)d.beta1, (double)d.t)));
    a.inv_c2 = d.t_device ? 0.0f : (float)(1.0 / (1.0 - std::pow((double)d.beta2, (double)d.t)));
    a.rate_device = d.rate_device; a.t_device = d.t_device; a.grad_scale_device = d.grad_scale_device; a.skip_device = d.skip_device;
    a.seed = d.seed; a.t = d.t; a.before = 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    int i = 0;
    for (; i < d.count; a.before += a.count) {
        a.count = 0;
        long long blocks = 0;
        for (; i < d.count && a.count < PXE_ADAMW_TENSORS_PER_LAUNCH; ++i) {
            const pxe_adamw_tensor& t = d.tensors[i];
            if (t.n == 0) continue;
            const long long mine = (t.n + kElements - 1) / kElements;
            if (blocks + mine > 0x3fffffffLL) break;       // (n <= 2^40 leaves room for one tensor)
            Entry& e = a.e[a.count++];
            e = {t.param, t.grad, t.m, t.v, t.m_scale, t.v_scale, t.master, t.n, (int)blocks, 0};
            const int per = psize == 4 ? 4 : 8;            // elements per access
            const uintptr_t wide = (uintptr_t)t.param | (uintptr_t)t.master | (small ? 0 : (uintptr_t)t.m | (uintptr_t)t.v);
            e.vector = wide % 16 == 0 && (uintptr_t)t.grad % std::min(16, per * gsize) == 0 && (!small || ((uintptr_t)t.m | (uintptr_t)t.v) % per == 0);
            blocks += mine;
        }
        if (a.count == 0) break;
        a.blocks = (int)blocks;
        int rc;
        if (d.param_type == PXE_F32)
            rc = d.grad_type == PXE_F32 ? launch<float, float>(s, a, small, master)
               : d.grad_type == PXE_BF16 ? launch<float, bf16>(s, a, small, master) : launch<float, f16>(s, a, small, master);
        else if (d.param_type == PXE_BF16)
            rc = d.grad_type == PXE_F32 ? launch<bf16, float>(s, a, small, master) : launch<bf16, bf16>(s, a, small, master);
        else
            rc = d.grad_type == PXE_F32 ? launch<f16, float>(s, a, small, master) : launch<f16, f16>(s, a, small, master);
        if (rc != PXE_OK) return rc;
    }
    return PXE_OK;
}
