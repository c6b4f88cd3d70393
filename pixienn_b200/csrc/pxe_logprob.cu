// Log probabilities of given classes, entropy and the largest alternatives of every row, and their gradient.
//
// With c = log2(e) / temperature, m = max x, d_j = (x_j - m) * c, S = sum 2^d_j, U = sum 2^d_j d_j:
//   logp = (x_target - m) / temperature - ln2 * log2 S,  entropy = ln2 * (log2 S - U / S),
//   dx_j = (g [j = target] - p_j (g + gH (ln p_j + entropy))) / temperature,  p_j = 2^(d_j - log2 S).
//
// The forward pass is bound by one read of the row: each thread keeps a running maximum with the sums S and U relative to
// it (both are rescaled when the maximum grows), and the threads' triples are joined at the end.  x - m is formed before
// the product with c, so that values near the maximum lose nothing and a row of the type's lowest value stays finite; d is
// held at -4096 (2^-4096 is 0), so that a probability of 0 adds 0 * d = 0 to U where x is -inf.
//
// The alternatives need no second pass over the row.  Keys order first by value (a NaN above everything), then by the
// lower class, and no two are equal.  Every thread keeps the largest key of its own elements; the k-th largest of those
// is a lower bound of the k-th largest of all, and whatever reaches it lies with the k threads of the largest keys.
// Only these k threads' elements are read again, and what reaches the bound (k and a few more) is ranked by counting.
#include <algorithm>

#include "pxe_types.cuh"

namespace pxe {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNoProbability = -4096.0f;
constexpr int kMaxTop = 32;
constexpr int kCandidates = 1024;

struct ProbsParams {
    const void* x;
    const void* target;
    float* logp;
    float* entropy;
    float* stats;
    float* top_logp;
    int* top_index;
    long long rows, inner, outer_stride, row_stride;
    int classes, target64, top;
    float c, inv_temperature;
};

struct ProbsBackParams {
    const void* x;
    const void* target;
    const float* stats;
    const float* dlogp;
    const float* dentropy;
    void* dx;
    long long rows, inner, outer_stride, row_stride, dx_outer_stride, dx_row_stride;
    int classes, target64, chunks;
    float c, inv_temperature;
};

__device__ __forceinline__ long long row_offset(long long row, long long inner, long long outer_stride, long long row_stride)
{
    const long long o = inner > 0 ? row / inner : 0;
    return o * outer_stride + (row - o * inner) * row_stride;
}

// The row's target: < 0 unused, >= classes out of range; rows without targets are used and have none.
__device__ __forceinline__ long long target_of(const void* target, int is64, long long row)
{
    return is64 ? gld(static_cast<const long long*>(target) + row) : (long long)gld(static_cast<const int*>(target) + row);
}

__device__ __forceinline__ float exp2_fast(float d) { return fast_ex2(d); }

// (maximum, S, U) of a part of a row
struct Part {
    float m, s, u;
};
__device__ __forceinline__ Part part_none() { return {-INFINITY, 0.0f, 0.0f}; }

// (x - m) * c, held at kNoProbability; a NaN stays one.  `m` is finite or NaN or +inf.
__device__ __forceinline__ float distance(float x, float m, float c) { return max_nan((x - m) * c, kNoProbability); }
__device__ __forceinline__ float origin(float m) { return m == -INFINITY ? 0.0f : m; }

// p's sums taken from the larger maximum m
__device__ __forceinline__ void rescale(Part& p, float m, float c)
{
    if (p.s == 0.0f) { p.m = m; return; }                  // nothing yet
    const float d = distance(p.m, m, c), r = exp2_fast(d);
    p.u = r * fmaf(p.s, d, p.u);
    p.s *= r;
    p.m = m;
}
__device__ __forceinline__ Part join(Part a, Part b, float c)
{
    const float m = max_nan(a.m, b.m), o = origin(m);
    rescale(a, o, c);
    rescale(b, o, c);
    return {m, a.s + b.s, a.u + b.u};
}

template <int N>
__device__ __forceinline__ void add_values(Part& p, const float (&x)[N], float c)
{
    float top = x[0];
#pragma unroll
    for (int j = 1; j < N; ++j) top = max_nan(top, x[j]);
    if (!(top <= p.m)) {                                   // larger, or NaN
        const float m = max_nan(p.m, top);
        rescale(p, origin(m), c);
        p.m = m;
    }
    const float o = origin(p.m);
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const float d = distance(x[j], o, c), e = exp2_fast(d);
        p.s += e;
        p.u = fmaf(e, d, p.u);
    }
}

// ---------------------------------------------------------------- keys of the alternatives
__device__ __forceinline__ uint32_t order_of(float x)
{
    if (x != x) return 0xffffffffu;
    const uint32_t b = __float_as_uint(x + 0.0f);          // -0 counts as 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t order)
{
    if (order == 0xffffffffu) return __int_as_float(0x7fffffff);
    return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
__device__ __forceinline__ unsigned long long key_of(float x, int index) { return (unsigned long long)order_of(x) << 32 | (uint32_t)~index; }
__device__ __forceinline__ int index_of(unsigned long long key) { return (int)~(uint32_t)key; }

// ---------------------------------------------------------------- forward: a block per row
// Elements of a row as the threads see them: `head` single elements up to the first 16-byte boundary, `nvec` vectors,
// and the rest.
template <typename T>
struct RowView {
    static constexpr int VEC = 16 / sizeof(T);
    const T* x;
    int head, nvec, classes;
    __device__ RowView(const T* row, int n) : x(row), classes(n)
    {
        const int off = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
        head = off ? min(VEC - off, n) : 0;
        nvec = (n - head) / VEC;
    }
    __device__ int tail() const { return head + nvec * VEC; }
};

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS)
log_probs_kernel(const ProbsParams p)
{
    constexpr int VEC = 16 / sizeof(T), WARPS = THREADS / 32;
    __shared__ Part parts[WARPS];
    __shared__ unsigned long long keys[THREADS], cand[kCandidates], best;
    __shared__ int slot[kMaxTop], n_cand;
    __shared__ float shared_l2s, shared_o;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const long long target = p.target ? target_of(p.target, p.target64, row) : 0;
        __syncthreads();
        if (target < 0) {
            if (t == 0) {
                gst(p.logp + row, 0.0f);
                if (p.entropy) gst(p.entropy + row, 0.0f);
                if (p.stats) { gst(p.stats + 3 * row, 0.0f); gst(p.stats + 3 * row + 1, 0.0f); gst(p.stats + 3 * row + 2, 0.0f); }
            }
            if (t < p.top) { gst(p.top_logp + row * p.top + t, 0.0f); gst(p.top_index + row * p.top + t, -1); }
            continue;
        }
        const RowView<T> r(static_cast<const T*>(p.x) + row_offset(row, p.inner, p.outer_stride, p.row_stride), p.classes);
        Part sum = part_none();
        float largest = -INFINITY;
        unsigned long long key = 0;                        // smaller than every element's
        auto single = [&](int i) {
            const float x[1] = {to_f32<T>(gld(r.x + i))};
            add_values<1>(sum, x, p.c);
            if (p.top) {
                const unsigned long long k = key_of(x[0], i);
                if (k > key) { key = k; largest = x[0]; }
            }
        };
        if (t < r.head) single(t);
        for (int v = t; v < r.nvec; v += THREADS) {
            float x[VEC];
            unpack<T, VEC>(gldv<Raw<T, VEC>>(r.x + r.head + v * VEC), x);
            add_values<VEC>(sum, x, p.c);
            if (p.top) {
                float m = x[0];
#pragma unroll
                for (int j = 1; j < VEC; ++j) m = max_nan(m, x[j]);
                if (!(m <= largest) || key == 0) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const unsigned long long k = key_of(x[j], r.head + v * VEC + j);
                        if (k > key) { key = k; largest = x[j]; }
                    }
                }
            }
        }
        if (r.tail() + t < p.classes) single(r.tail() + t);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            Part other;
            other.m = __shfl_xor_sync(0xffffffffu, sum.m, o);
            other.s = __shfl_xor_sync(0xffffffffu, sum.s, o);
            other.u = __shfl_xor_sync(0xffffffffu, sum.u, o);
            sum = join(sum, other, p.c);
        }
        if (lane == 0) parts[warp] = sum;
        if (p.top) {
            keys[t] = key;
            if (t == 0) n_cand = 0;
        }
        __syncthreads();
        if (t == 0) {
            for (int w = 1; w < WARPS; ++w) sum = join(sum, parts[w], p.c);
            const float o = origin(sum.m), l2s = log2f(sum.s);             // a row of -inf: S = 0
            const float entropy = sum.s == 0.0f ? 0.0f : kLn2 * (l2s - sum.u / sum.s);
            if (p.logp) {
                float logp = __int_as_float(0x7fffffff);
                if (target < p.classes) {
                    const float x = to_f32<T>(gld(r.x + target));
                    logp = sum.s == 0.0f || x == -INFINITY ? (sum.s != sum.s ? sum.s : -INFINITY) : (x - o) * p.inv_temperature - kLn2 * l2s;
                }
                gst(p.logp + row, logp);
            }
            if (p.entropy) gst(p.entropy + row, entropy);
            if (p.stats) { gst(p.stats + 3 * row, o); gst(p.stats + 3 * row + 1, l2s); gst(p.stats + 3 * row + 2, entropy); }
            shared_l2s = l2s;
            shared_o = o;
        }
        if (p.top == 0) continue;
        const int top = p.top;
        // the rank of this thread's key among the threads'; the threads of the `top` largest
        if (t < kMaxTop) slot[t] = -1;
        __syncthreads();
        int rank = 0;
        for (int i = 0; i < THREADS; ++i) rank += keys[i] > key;
        if (key != 0 && rank < top) slot[rank] = t;
        __syncthreads();
        const unsigned long long bound = slot[top - 1] >= 0 ? keys[slot[top - 1]] : 0;
        // visit(k) for every element's key of the slots' threads, a warp for each slot
        auto visit_slots = [&](auto&& visit) {
            for (int s = warp; s < top; s += WARPS) {
                const int owner = slot[s];
                if (owner < 0) break;
                if (lane == 0 && owner < r.head) visit(key_of(to_f32<T>(gld(r.x + owner)), owner));
                for (int v = owner + lane * THREADS; v < r.nvec; v += 32 * THREADS) {
                    float x[VEC];
                    unpack<T, VEC>(gldv<Raw<T, VEC>>(r.x + r.head + v * VEC), x);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) visit(key_of(x[j], r.head + v * VEC + j));
                }
                const int i = r.tail() + owner;
                if (lane == 0 && i < p.classes) visit(key_of(to_f32<T>(gld(r.x + i)), i));
            }
        };
        visit_slots([&](unsigned long long k) {
            if (k >= bound) {
                const int at = atomicAdd(&n_cand, 1);
                if (at < kCandidates) cand[at] = k;
            }
        });
        __syncthreads();
        const float l2s = shared_l2s, o = shared_o;
        auto store = [&](int place, unsigned long long k) {
            const float x = value_of((uint32_t)(k >> 32));
            const float logp = l2s == -INFINITY || (x == -INFINITY && l2s == l2s) ? -INFINITY : (x - o) * p.inv_temperature - kLn2 * l2s;
            gst(p.top_logp + row * top + place, logp);
            gst(p.top_index + row * top + place, index_of(k));
        };
        const int n = n_cand;
        if (n <= kCandidates) {
            for (int i = t; i < n; i += THREADS) {
                const unsigned long long k = cand[i];
                int place = 0;
                for (int j = 0; j < n; ++j) place += cand[j] > k;
                if (place < top) store(place, k);
            }
        } else {                                           // the k threads hold more large values than the list: one after the other
            unsigned long long last = ~0ull;
            for (int place = 0; place < top; ++place) {
                if (t == 0) best = 0;
                __syncthreads();
                unsigned long long mine = 0;
                visit_slots([&](unsigned long long k) { if (k < last && k > mine) mine = k; });
                atomicMax(&best, mine);
                __syncthreads();
                last = best;
                if (t == 0) store(place, last);
                __syncthreads();
            }
        }
    }
}

// ---------------------------------------------------------------- backward
// `chunks` blocks per row.  Vectors where x and dx have the same distance from a 16-byte boundary, else single elements.
template <typename T>
__global__ void __launch_bounds__(256)
log_probs_backward_kernel(const ProbsBackParams p)
{
    constexpr int VEC = 16 / sizeof(T);
    const long long row = blockIdx.x / p.chunks;
    const int chunk = (int)(blockIdx.x - row * p.chunks);
    const T* x = static_cast<const T*>(p.x) + row_offset(row, p.inner, p.outer_stride, p.row_stride);
    T* dx = static_cast<T*>(p.dx) + row_offset(row, p.inner, p.dx_outer_stride, p.dx_row_stride);
    const long long target = p.target ? target_of(p.target, p.target64, row) : 0;
    const float o = gld(p.stats + 3 * row), l2s = gld(p.stats + 3 * row + 1), entropy = gld(p.stats + 3 * row + 2);
    const bool used = target >= 0 && l2s != -INFINITY;
    float g = 0.0f;
    if (p.dlogp && p.target) g = target < p.classes ? gld(p.dlogp + row) : __int_as_float(0x7fffffff);
    const float gh = p.dentropy ? gld(p.dentropy + row) : 0.0f;
    // dx = p * (a + b * d), and g / T more at the target
    const float a = -(g + gh * (entropy - kLn2 * l2s)) * p.inv_temperature, b = -gh * kLn2 * p.inv_temperature;
    const float inv_s = exp2f(-l2s), at_target = g * p.inv_temperature;
    auto gradient = [&](float v, int i) {
        const float d = distance(v, o, p.c);
        const float q = exp2_fast(d) * inv_s * fmaf(b, d, a);
        return p.target && i == target ? q + at_target : q;
    };
    const RowView<T> r(x, p.classes);
    const bool same = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15) == 0;
    const int threads = blockDim.x * p.chunks, t = chunk * blockDim.x + threadIdx.x;
    auto single = [&](int i) { gst(dx + i, from_f32<T>(used ? gradient(to_f32<T>(gld(x + i)), i) : 0.0f)); };
    if (!same) {
        for (int i = t; i < p.classes; i += threads) single(i);
        return;
    }
    if (t < r.head) single(t);
    for (int v = t; v < r.nvec; v += threads) {
        const int i = r.head + v * VEC;
        float f[VEC];
        if (used) {
            unpack<T, VEC>(gldv<Raw<T, VEC>>(x + i), f);
#pragma unroll
            for (int j = 0; j < VEC; ++j) f[j] = gradient(f[j], i + j);
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) f[j] = 0.0f;
        }
        gstv(dx + i, pack<T, VEC>(f));
    }
    if (r.tail() + t < p.classes) single(r.tail() + t);
}

// ---------------------------------------------------------------- host
// Rows of x or dx: the checked strides, and the span they cover as one row tensor.
int check_rows(const char* name, const void* ptr, int size, long long rows, long long& inner, long long& outer, long long& stride, int classes)
{
    PXE_REQUIRE(reinterpret_cast<uintptr_t>(ptr) % size == 0, "%s is not aligned to its elements", name);
    if (inner == 0) { inner = rows; outer = 0; }
    if (stride == 0) stride = classes;
    PXE_REQUIRE(inner > 0 && rows % inner == 0, "%s: %lld rows in groups of %lld", name, rows, inner);
    PXE_REQUIRE(stride >= classes, "%s: row stride %lld is less than %d classes", name, stride, classes);
    PXE_REQUIRE(rows == inner || outer >= (inner - 1) * stride + classes, "%s: outer stride %lld, a group covers %lld", name, outer, (inner - 1) * stride + classes);
    return PXE_OK;
}
RowSpan group_span(const void* ptr, int size, long long rows, long long inner, long long outer, long long stride, int classes)
{
    return {ptr, rows / inner, outer * size, ((inner - 1) * stride + classes) * size};
}

}  // namespace
}  // namespace pxe

using namespace pxe;

extern "C" int pxe_log_probs(pxe_stream_t stream, const pxe_log_probs_desc* dp)
{
    PXE_REQUIRE(dp != nullptr, "log_probs: null descriptor");
    const pxe_log_probs_desc& d = *dp;
    PXE_REQUIRE(valid_dtype(d.type), "log_probs: unknown type %d", d.type);
    PXE_REQUIRE(d.rows >= 0 && d.classes > 0, "log_probs: shape [%lld, %d]", d.rows, d.classes);
    PXE_REQUIRE(d.rows <= 0x7fffffffLL, "log_probs: too many rows");
    PXE_REQUIRE(d.classes <= (1 << 30), "log_probs: too many classes");
    PXE_REQUIRE(d.temperature > 0.0f && d.temperature < INFINITY, "log_probs: temperature is not a positive number");
    PXE_REQUIRE(d.top >= 0 && d.top <= kMaxTop && d.top <= d.classes, "log_probs: top %d is not in 0..%d or above %d classes", d.top, kMaxTop, d.classes);
    if (d.rows == 0) return PXE_OK;
    PXE_REQUIRE(d.x != nullptr, "log_probs: x is null");
    PXE_REQUIRE((d.target != nullptr) == (d.logp != nullptr), "log_probs: target and logp come together");
    PXE_REQUIRE((d.top > 0) == (d.top_logp != nullptr) && (d.top > 0) == (d.top_index != nullptr), "log_probs: top_logp and top_index come with top > 0");
    ProbsParams p{};
    p.x = d.x; p.target = d.target; p.logp = d.logp; p.entropy = d.entropy; p.stats = d.stats; p.top_logp = d.top_logp; p.top_index = d.top_index;
    p.rows = d.rows; p.inner = d.inner; p.outer_stride = d.outer_stride; p.row_stride = d.row_stride;
    p.classes = d.classes; p.target64 = d.target_is_int64; p.top = d.top; p.c = kLog2e / d.temperature; p.inv_temperature = 1.0f / d.temperature;
    const int size = dtype_bytes(d.type);
    { const int rc = check_rows("log_probs: x", d.x, size, d.rows, p.inner, p.outer_stride, p.row_stride, d.classes); if (rc != PXE_OK) return rc; }
    const RowSpan x = group_span(d.x, size, d.rows, p.inner, p.outer_stride, p.row_stride, d.classes);
    const struct { const void* ptr; long long bytes; } outs[] = {{d.logp, d.rows * 4}, {d.entropy, d.rows * 4}, {d.stats, d.rows * 12},
                                                                 {d.top_logp, d.rows * d.top * 4}, {d.top_index, d.rows * d.top * 4}};
    for (const auto& o : outs)
        PXE_REQUIRE(!o.ptr || (o.ptr != d.x && o.ptr != d.target && !rows_conflict({o.ptr, 1, 0, o.bytes}, x)), "log_probs: an output overlaps an input");
    DeviceInfo di;
    { const int rc = device_info(&di); if (rc != PXE_OK) return rc; }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const unsigned grid = (unsigned)d.rows;
    if (d.type == PXE_F32) log_probs_kernel<float, 512><<<grid, 512, 0, s>>>(p);
    else if (d.type == PXE_BF16) log_probs_kernel<bf16, 512><<<grid, 512, 0, s>>>(p);
    else log_probs_kernel<f16, 512><<<grid, 512, 0, s>>>(p);
    PXE_LAUNCH_OK("log_probs_kernel");
    return PXE_OK;
}

extern "C" int pxe_log_probs_backward(pxe_stream_t stream, const pxe_log_probs_backward_desc* dp)
{
    PXE_REQUIRE(dp != nullptr, "log_probs_backward: null descriptor");
    const pxe_log_probs_backward_desc& d = *dp;
    PXE_REQUIRE(valid_dtype(d.type), "log_probs_backward: unknown type %d", d.type);
    PXE_REQUIRE(d.rows >= 0 && d.classes > 0, "log_probs_backward: shape [%lld, %d]", d.rows, d.classes);
    PXE_REQUIRE(d.classes <= (1 << 30), "log_probs_backward: too many classes");
    PXE_REQUIRE(d.temperature > 0.0f && d.temperature < INFINITY, "log_probs_backward: temperature is not a positive number");
    if (d.rows == 0) return PXE_OK;
    PXE_REQUIRE(d.x && d.stats && d.dx, "log_probs_backward: null pointer");
    PXE_REQUIRE((d.dlogp && d.target) || d.dentropy, "log_probs_backward: neither dlogp with target nor dentropy");
    PXE_REQUIRE(!d.dlogp || d.target, "log_probs_backward: dlogp without target");
    ProbsBackParams p{};
    p.x = d.x; p.target = d.target; p.stats = d.stats; p.dlogp = d.dlogp; p.dentropy = d.dentropy; p.dx = d.dx;
    p.rows = d.rows; p.inner = d.inner; p.outer_stride = d.outer_stride; p.row_stride = d.row_stride;
    p.dx_outer_stride = d.dx_outer_stride; p.dx_row_stride = d.dx_row_stride;
    p.classes = d.classes; p.target64 = d.target_is_int64;
    p.c = kLog2e / d.temperature; p.inv_temperature = 1.0f / d.temperature;
    const int size = dtype_bytes(d.type);
    long long inner = d.inner;
    { const int rc = check_rows("log_probs_backward: x", d.x, size, d.rows, p.inner, p.outer_stride, p.row_stride, d.classes); if (rc != PXE_OK) return rc; }
    { const int rc = check_rows("log_probs_backward: dx", d.dx, size, d.rows, inner, p.dx_outer_stride, p.dx_row_stride, d.classes); if (rc != PXE_OK) return rc; }
    const RowSpan x = group_span(d.x, size, d.rows, p.inner, p.outer_stride, p.row_stride, d.classes);
    const RowSpan dx = group_span(d.dx, size, d.rows, inner, p.dx_outer_stride, p.dx_row_stride, d.classes);
    PXE_REQUIRE(d.dx == d.x ? p.row_stride == p.dx_row_stride && p.outer_stride == p.dx_outer_stride : !rows_conflict(dx, x),
                "log_probs_backward: dx partially overlaps x");
    const struct { const void* ptr; long long bytes; } ins[] = {{d.stats, d.rows * 12}, {d.dlogp, d.rows * 4}, {d.dentropy, d.rows * 4},
                                                                {d.target, d.rows * (d.target_is_int64 ? 8 : 4)}};
    for (const auto& i : ins)
        PXE_REQUIRE(!i.ptr || (i.ptr != d.dx && !rows_conflict({i.ptr, 1, 0, i.bytes}, dx)), "log_probs_backward: dx overlaps an input");
    p.chunks = std::max(1, (d.classes + 256 * 32 - 1) / (256 * 32));
    PXE_REQUIRE(d.rows * p.chunks <= 0x7fffffffLL, "log_probs_backward: too many rows");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const unsigned grid = (unsigned)(d.rows * p.chunks);
    if (d.type == PXE_F32) log_probs_backward_kernel<float><<<grid, 256, 0, s>>>(p);
    else if (d.type == PXE_BF16) log_probs_backward_kernel<bf16><<<grid, 256, 0, s>>>(p);
    else log_probs_backward_kernel<f16><<<grid, 256, 0, s>>>(p);
    PXE_LAUNCH_OK("log_probs_backward_kernel");
    return PXE_OK;
}
