// Log probabilities of given classes, entropy and the largest alternatives of every row, and their gradient.
//
// With c = log2(e) / temperature, m = max x, d_j = (x_j - m) * c, S = sum 2^d_j, U = sum 2^d_j d_j:
//   logp = (x_target - m) / temperature - ln2 * log2 S,  entropy = ln2 * (log2 S - U / S),
//   dx_j = (g [j = target] - p_j (g + gH (ln p_j + entropy))) / temperature,  p_j = 2^(d_j - log2 S).
//
// The forward pass is bound by one read of the row, and next to it by issue: at the memory's rate a 16-bit row leaves 11
// issue slots an element on an SM.  Each thread takes four 16-byte vectors at a time, finds their maximum (two elements
// an instruction in 16 bits), rescales its sums only when the running maximum grows, and forms d = x * c - o with one
// rounding from the origin o = fl(m * c), two elements an instruction (as S and U).  The origin's rounding is the same
// shift for every element, up to half a unit of o, and is taken out of log2 S at the end: at |m c| <= 2^24 it is at most
// 1/2.  Beyond, 2^shift would leave the range of a float (at m = -1e10 and temperature 1 the shift is 440).  A row whose own
// maximum lies beyond +-2^24 / c is therefore read again with (x - m) * c, which neither overflows nor loses the row; and
// partial sums under a maximum of m c < -2^25, which count for nothing in any other row (a mask's finite value, until the
// thread or another one meets more), take the origin 0, from which all they hold adds 0.  Values of -inf are held at -2^100
// (the lowest value in fp16), so that a probability of 0 adds 0 * d = 0 to U; what they count for is nothing only from
// further away, so that a row in fp16 under half the lowest value, and every row at temperatures above 72 or below 1e-7, is
// read again as well.
//
// The alternatives need no second pass over the row.  The k-th largest of the threads' own maxima is a lower bound of the
// k-th largest value of all, and whatever reaches it lies with the threads whose maximum does: k of them, and those that
// tie.  Only these threads' elements are read again, and what reaches the bound (k and a few more) is ranked by counting
// on keys that order first by value (a NaN above everything), then by the lower class.  Where more threads tie than the
// list holds (a row with fewer than k values that are not -inf), every thread finds the largest key of its own elements
// first; keys are unique, so that exactly k threads are left.
//
// Few rows leave most SMs idle, so a long row is then split over a cluster of up to eight blocks, which exchange their
// sums and their alternatives through distributed shared memory; short rows take a warp or eight lanes of one each and
// stay in registers, many rows of middling length a small block each.
#include <cooperative_groups.h>

#include <algorithm>

#include "pxe_types.cuh"

namespace pxe {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNoProbability = -4096.0f;
constexpr int kMaxTop = 32;

struct ProbsParams {
    const void* x;
    const void* target;
    float* logp;
    float* entropy;
    float* stats;
    float* top_logp;
    int* top_index;
    long long rows, inner, outer_stride, row_stride;
    int classes, target64, top, cluster, careful;
    float c, inv_temperature, far;                         // far = kFar / c
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

// Where a row begins.  Rows are less than 2^31 and inner at most rows, so that 32 bits would do for the division; they are
// used where short rows share a block (65536 x 80 fp32).  Where a block has one row the division counts for nothing, but
// its result then stays in registers that the sums need (4095 x 50003 bf16: 77 us, 20 bytes spilled, against 71).
template <typename INT>
__device__ __forceinline__ long long row_offset(long long row, long long inner, long long outer_stride, long long row_stride)
{
    const long long o = (INT)row / (INT)inner;
    return o * outer_stride + (row - o * inner) * row_stride;
}

// The row's target: < 0 unused, >= classes out of range; rows without targets are used and have none.
__device__ __forceinline__ long long target_of(const void* target, int is64, long long row)
{
    return is64 ? gld(static_cast<const long long*>(target) + row) : (long long)gld(static_cast<const int*>(target) + row);
}

__device__ __forceinline__ float exp2_fast(float d) { return fast_ex2(d); }

// (x - m) * c, held at kNoProbability; a NaN stays one.  `m` is finite or NaN or +inf.
__device__ __forceinline__ float distance(float x, float m, float c) { return max_nan((x - m) * c, kNoProbability); }

// ---------------------------------------------------------------- sums of a part of a row
// The maximum m and the sums S and U from the origin o = origin_of(m, c).
struct Part {
    float m, s, u;
};
constexpr float kFar = 16777216.0f;                        // of a row's m * c; its rounding is up to a half, and 1 at twice that
// (a product that is never contracted into what uses it: the origin's rounding has to be the same everywhere)
__device__ __forceinline__ float origin_of(float m, float c)
{
    const float o = __fmul_rn(m, c);
    return o < -2.0f * kFar ? 0.0f : o;                    // (2^-kFar of a row that is not read again)
}

__device__ __forceinline__ void rescale(float& s, float& u, float from, float to)
{
    if (s == 0.0f) return;                                 // nothing yet
    const float d = from - to, r = exp2_fast(d);
    u = r * fmaf(s, d, u);
    s *= r;
}
__device__ __forceinline__ Part join(Part a, Part b, float c)
{
    const float m = max_nan(a.m, b.m), o = origin_of(m, c);
    rescale(a.s, a.u, origin_of(a.m, c), o);
    rescale(b.s, b.u, origin_of(b.m, c), o);
    return {m, a.s + b.s, a.u + b.u};
}

// 32-bit words of a vector: one float or two 16-bit elements each.  LOW, low: what -inf is held at; a row whose maximum is
// under `lowest` is too near to that and read again (in 32 bits and bf16 such a row is beyond -2^24 / c already).
template <typename T> struct Word;
template <> struct Word<float> {
    static constexpr uint32_t LOW = 0xf1800000u, NONE = 0xff800000u;               // -2^100, -inf
    static constexpr float low = -0x1p100f, lowest = -INFINITY;
    static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b) { return __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b))); }
    static __device__ __forceinline__ float largest(uint32_t a) { return __uint_as_float(a); }
};
template <> struct Word<bf16> {
    static constexpr uint32_t LOW = 0xf180f180u, NONE = 0xff80ff80u;               // -2^100, -inf
    static constexpr float low = -0x1p100f, lowest = -INFINITY;
    static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b)
    {
        uint32_t r;
        asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ float largest(uint32_t a) { float x, y; split<bf16>(a, x, y); return max_nan(x, y); }
};
template <> struct Word<f16> {
    static constexpr uint32_t LOW = 0xfbfffbffu, NONE = 0xfc00fc00u;               // -65504, -inf
    static constexpr float low = -65504.0f, lowest = -32752.0f;
    static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b)
    {
        uint32_t r;
        asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ float largest(uint32_t a) { float x, y; split<f16>(a, x, y); return max_nan(x, y); }
};

constexpr int kBatch = 4;                                  // vectors a thread takes at a time

// A thread's sums: S and U as two halves each (even and odd elements), from the origin o.
struct Running {
    float m, o;
    unsigned long long s, u;
    __device__ __forceinline__ void clear() { m = -INFINITY; o = 0.0f; s = u = pair(0.0f, 0.0f); }
    __device__ __forceinline__ void grow(float largest, float c)
    {
        if (largest <= m) return;                          // (a NaN is not)
        m = max_nan(m, largest);
        const float to = origin_of(m, c);
        float s0, s1, u0, u1;
        unpair(s, s0, s1);
        unpair(u, u0, u1);
        rescale(s0, u0, o, to);
        rescale(s1, u1, o, to);
        s = pair(s0, s1);
        u = pair(u0, u1);
        o = to;
    }
    __device__ __forceinline__ void add(float x, float y, unsigned long long c2, unsigned long long o2)
    {
        const unsigned long long d = fma2(pair(x, y), c2, o2);
        float d0, d1;
        unpair(d, d0, d1);
        const unsigned long long e = pair(exp2_fast(d0), exp2_fast(d1));
        s = add2(s, e);
        u = fma2(e, d, u);
    }
    // one element in the first half, nothing in the other
    __device__ __forceinline__ void add_one(float x, float low, float c)
    {
        grow(x, c);
        const float d = fmaf(max_nan(x, low), c, -o), e = exp2_fast(d);
        s = add2(s, pair(e, 0.0f));
        u = add2(u, pair(e * d, 0.0f));
    }
    // N vectors
    template <typename T, int N>
    __device__ __forceinline__ void add_vectors(uint4* raw, float c)
    {
        uint32_t* w = reinterpret_cast<uint32_t*>(raw);
        uint32_t top = w[0];
#pragma unroll
        for (int k = 1; k < 4 * N; ++k) top = Word<T>::max(top, w[k]);
        grow(Word<T>::largest(top), c);
        const unsigned long long c2 = pair(c, c), o2 = pair(-o, -o);
#pragma unroll
        for (int k = 0; k < 4 * N; ++k) w[k] = Word<T>::max(w[k], Word<T>::LOW);
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int k = 0; k < 2 * N; ++k) add(__uint_as_float(w[2 * k]), __uint_as_float(w[2 * k + 1]), c2, o2);
        } else {
#pragma unroll
            for (int k = 0; k < 4 * N; ++k) {
                float x, y;
                split<T>(w[k], x, y);
                add(x, y, c2, o2);
            }
        }
    }
    __device__ __forceinline__ Part part() const
    {
        float s0, s1, u0, u1;
        unpair(s, s0, s1);
        unpair(u, u0, u1);
        return {m, s0 + s1, u0 + u1};
    }
};

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

// ---------------------------------------------------------------- forward
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
    __device__ int element(int v) const { return head + v * VEC; }
};

__device__ __forceinline__ float warp_max(float v)
{
    float r;
    asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ void warp_sum(float& a, float& b)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
    }
}

// The block's part from its threads': the maximum first, so that every thread rescales once.  All get the result.
template <int THREADS>
__device__ __forceinline__ Part join_block(Part p, Part* parts, float c)
{
    constexpr int WARPS = THREADS / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float m = warp_max(p.m);
    rescale(p.s, p.u, origin_of(p.m, c), origin_of(m, c));
    warp_sum(p.s, p.u);
    if (lane == 0) parts[warp] = {m, p.s, p.u};
    __syncthreads();
    p = lane < WARPS ? parts[lane] : Part{-INFINITY, 0.0f, 0.0f};
    const float all = warp_max(p.m);
    rescale(p.s, p.u, origin_of(p.m, c), origin_of(all, c));
    warp_sum(p.s, p.u);
    p.m = all;
    __syncthreads();
    return p;
}

// How many of `n` keys, in descending order, are larger than `key`.
__device__ __forceinline__ int larger_than(const unsigned long long* sorted, int n, unsigned long long key)
{
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (sorted[mid] > key) lo = mid + 1; else hi = mid;
    }
    return lo;
}

// Descending order over the lanes of a warp: a bitonic sort, and the last merge of one.
template <int STEP>
__device__ __forceinline__ uint32_t merge_descending(uint32_t v)
{
#pragma unroll
    for (int step = STEP; step > 0; step >>= 1) {
        const uint32_t other = __shfl_xor_sync(0xffffffffu, v, step);
        v = (threadIdx.x & step) == 0 ? max(v, other) : min(v, other);
    }
    return v;
}
__device__ __forceinline__ uint32_t sort_descending(uint32_t v)
{
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1) {
#pragma unroll
        for (int step = size >> 1; step > 0; step >>= 1) {
            const uint32_t other = __shfl_xor_sync(0xffffffffu, v, step);
            v = ((lane & step) == 0) == ((lane & size) == 0) ? max(v, other) : min(v, other);
        }
    }
    return v;
}

constexpr int kCandidates = 1024;                          // of a block
// Of 256 threads on an SM: 32 registers a thread, and no loads ahead (4095 x 50003 bf16 71 us, at six blocks 73, at four 83).
constexpr int kBlocks = 8;
constexpr int kSelected = 64;                              // threads of a block whose elements are read again

template <int THREADS>
struct TopShared {
    uint32_t maxima[THREADS / 32][32];
    unsigned long long keys[THREADS];                      // every warp's in descending order
    unsigned long long cand[kCandidates];
    unsigned long long list[kMaxTop];                      // the block's alternatives in order
    unsigned long long best;
    int selected[kSelected], n_selected, n_cand;
};
struct NoTop {};

// What a block takes of a row: the vectors [v0, v1), and the single elements in front and behind.
template <typename T>
struct Slice {
    RowView<T> r;
    int v0, v1;
    bool head, tail;
    // visit(key) for every element of thread `who` of THREADS; `first` of `step` visitors
    template <int THREADS, typename F>
    __device__ __forceinline__ void visit(int who, int first, int step, F&& f) const
    {
        constexpr int VEC = RowView<T>::VEC;
        for (int v = v0 + who + first * THREADS; v < v1; v += step * THREADS) {
            float x[VEC];
            unpack<T, VEC>(gldv<Raw<T, VEC>>(r.x + r.element(v)), x);
#pragma unroll
            for (int j = 0; j < VEC; ++j) f(key_of(x[j], r.element(v) + j));
        }
        if (first == 0) {
            if (head && who < r.head) f(key_of(to_f32<T>(gld(r.x + who)), who));
            const int i = r.tail() + who;
            if (tail && i < r.classes) f(key_of(to_f32<T>(gld(r.x + i)), i));
        }
    }
};

// sh.cand in order into sh.list
template <int THREADS>
__device__ __forceinline__ void rank_candidates(TopShared<THREADS>& sh, int n, int top)
{
    for (int i = threadIdx.x; i < n; i += THREADS) {
        const unsigned long long mine = sh.cand[i];
        int place = 0;
        for (int j = 0; j < n; ++j) place += sh.cand[j] > mine;
        if (place < top) sh.list[place] = mine;
    }
}

// The `top` largest keys of a slice into sh.list (0 where there are fewer).  largest: order_of this thread's maximum, 0
// where it has no element.
template <typename T, int THREADS>
__device__ __forceinline__ void block_top(TopShared<THREADS>& sh, const Slice<T>& s, uint32_t largest, int top)
{
    constexpr int WARPS = THREADS / 32;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    // the 32 largest of the threads' maxima: sorted by warp, then merged two lists at a time
    sh.maxima[warp][lane] = sort_descending(largest);
    if (t < kMaxTop) sh.list[t] = 0;
    if (t == 0) sh.n_cand = sh.n_selected = 0;
#pragma unroll
    for (int w = WARPS / 2; w > 0; w >>= 1) {
        __syncthreads();
        if (warp < w) sh.maxima[warp][lane] = merge_descending<16>(max(sh.maxima[warp][lane], sh.maxima[warp + w][31 - lane]));
    }
    __syncthreads();
    const uint32_t least = sh.maxima[0][top - 1];
    if (largest != 0 && largest >= least) {
        const int at = atomicAdd(&sh.n_selected, 1);
        if (at < kSelected) sh.selected[at] = t;
    }
    __syncthreads();
    const int n_selected = sh.n_selected;
    auto offer = [&](unsigned long long key, unsigned long long bound) {
        if (key >= bound) {
            const int at = atomicAdd(&sh.n_cand, 1);
            if (at < kCandidates) sh.cand[at] = key;
        }
    };
    if (n_selected <= kSelected) {
        const int per = max(1, (s.v1 - s.v0 + THREADS - 1) / THREADS);            // visitors for each thread, a vector each
        for (int i = t; i < n_selected * per; i += THREADS)
            s.template visit<THREADS>(sh.selected[i / per], i % per, per, [&](unsigned long long key) { offer(key, (unsigned long long)least << 32); });
        __syncthreads();
        if (sh.n_cand <= kCandidates) {
            rank_candidates(sh, sh.n_cand, top);
            __syncthreads();
            return;
        }
    }
    // every thread's largest key; the threads of the `top` largest
    unsigned long long key = 0;
    s.template visit<THREADS>(t, 0, 1, [&](unsigned long long k) { key = k > key ? k : key; });
    int owner = t;
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1) {
#pragma unroll
        for (int step = size >> 1; step > 0; step >>= 1) {
            const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, step);
            const int other_owner = __shfl_xor_sync(0xffffffffu, owner, step);
            const bool keep_larger = ((lane & step) == 0) == ((lane & size) == 0);
            if (keep_larger ? other > key : other < key) { key = other; owner = other_owner; }
        }
    }
    __syncthreads();
    sh.keys[t] = key;
    if (t < kMaxTop) sh.selected[t] = -1;
    if (t == 0) sh.n_cand = 0;
    __syncthreads();
    if (key != 0 && lane < top) {
        int rank = lane;
        for (int w = 0; w < WARPS; ++w)
            if (w != warp) rank += larger_than(sh.keys + 32 * w, top, key);
        if (rank < top) { sh.selected[rank] = owner; if (rank == top - 1) sh.best = key; }
    }
    __syncthreads();
    const unsigned long long bound = sh.selected[top - 1] >= 0 ? sh.best : 0;
    auto visit_selected = [&](auto&& f) {                  // a warp for each
        for (int k = warp; k < top && sh.selected[k] >= 0; k += WARPS) s.template visit<THREADS>(sh.selected[k], lane, 32, f);
    };
    visit_selected([&](unsigned long long k) { offer(k, bound); });
    __syncthreads();
    if (sh.n_cand <= kCandidates) {
        rank_candidates(sh, sh.n_cand, top);
    } else {                                               // they hold more large values than the list: one after the other
        unsigned long long last = ~0ull;
        for (int place = 0; place < top; ++place) {
            if (t == 0) sh.best = 0;
            __syncthreads();
            unsigned long long mine = 0;
            visit_selected([&](unsigned long long k) { if (k < last && k > mine) mine = k; });
            atomicMax(&sh.best, mine);
            __syncthreads();
            last = sh.best;
            if (t == 0) sh.list[place] = last;
            __syncthreads();
        }
    }
    __syncthreads();
}

// What a row's sums say: the maximum (0 for a row of -inf), S, U / S and log2 S from that maximum.
struct RowResult {
    float m, s, mean, l2s;
};
__device__ __forceinline__ float logp_of(const RowResult& a, float x, const ProbsParams& p)
{
    if (a.s == 0.0f || (x == -INFINITY && a.s == a.s)) return -INFINITY;
    return (x - a.m) * p.inv_temperature - kLn2 * a.l2s;
}
template <typename T>
__device__ __forceinline__ void store_row(const ProbsParams& p, long long row, long long target, const T* x, const RowResult& a, float log2_s)
{
    const float entropy = a.s == 0.0f ? 0.0f : kLn2 * (log2_s - a.mean);
    if (p.logp) gst(p.logp + row, target < p.classes ? logp_of(a, to_f32<T>(gld(x + target)), p) : __int_as_float(0x7fffffff));
    if (p.entropy) gst(p.entropy + row, entropy);
    if (p.stats) { gst(p.stats + 3 * row, a.m); gst(p.stats + 3 * row + 1, a.s == 0.0f ? -INFINITY : a.l2s); gst(p.stats + 3 * row + 2, entropy); }
}
// A row without use; `t` of at least kMaxTop threads.
__device__ __forceinline__ void store_unused(const ProbsParams& p, long long row, int t)
{
    if (t == 0) {
        gst(p.logp + row, 0.0f);
        if (p.entropy) gst(p.entropy + row, 0.0f);
        if (p.stats) { gst(p.stats + 3 * row, 0.0f); gst(p.stats + 3 * row + 1, 0.0f); gst(p.stats + 3 * row + 2, 0.0f); }
    }
    if (t < p.top) { gst(p.top_logp + row * p.top + t, 0.0f); gst(p.top_index + row * p.top + t, -1); }
}
__device__ __forceinline__ void store_top(const ProbsParams& p, long long row, int place, unsigned long long key, const RowResult& a)
{
    gst(p.top_logp + row * p.top + place, logp_of(a, value_of((uint32_t)(key >> 32)), p));
    gst(p.top_index + row * p.top + place, index_of(key));
}

// A row to a block (or to a cluster of them, a part of it each).  4095 x 50003 bf16: 71 us, 0.89 of the copy rate on rows
// that begin at any alignment, bound by issue (0.69 of the slots, and the exponentials' unit at 0.64); 20 alternatives: 94 us.
template <typename T, int THREADS, bool TOP, bool CLUSTER>
__global__ void __launch_bounds__(THREADS, kBlocks * 256 / THREADS)
log_probs_kernel(const ProbsParams p)
{
    constexpr int VEC = RowView<T>::VEC;
    namespace cg = cooperative_groups;
    __shared__ Part parts[THREADS / 32];
    __shared__ Part shared_part;
    __shared__ std::conditional_t<TOP, TopShared<THREADS>, NoTop> sh;
    __shared__ std::conditional_t<TOP && CLUSTER, unsigned long long[8 * kMaxTop], NoTop> lists;
    const int t = threadIdx.x;
    const int ranks = CLUSTER ? p.cluster : 1, rank = CLUSTER ? (int)(blockIdx.x % p.cluster) : 0;
    const long long row = blockIdx.x / ranks;
    const long long target = p.target ? target_of(p.target, p.target64, row) : 0;
    if (target < 0) {
        if (rank == 0) store_unused(p, row, t);
        return;
    }
    const long long offset = row_offset<long long>(row, p.inner, p.outer_stride, p.row_stride);
    Slice<T> s{RowView<T>(static_cast<const T*>(p.x) + offset, p.classes), 0, 0, rank == 0, rank == ranks - 1};
    const RowView<T>& r = s.r;
    const int per = (r.nvec + ranks - 1) / ranks;
    s.v0 = min(rank * per, r.nvec);
    s.v1 = min(s.v0 + per, r.nvec);
    Running sum;
    sum.clear();
    for (int first = s.v0; first < s.v1; first += kBatch * THREADS) {
        uint4 raw[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            constexpr uint32_t none = Word<T>::NONE;
            raw[k] = make_uint4(none, none, none, none);
            if (first + t + k * THREADS < s.v1) raw[k] = gldv<uint4>(r.x + r.element(first + t + k * THREADS));
        }
        if (first + kBatch * THREADS <= s.v1) {
            sum.template add_vectors<T, kBatch>(raw, p.c);
        } else {                                       // the slice's last vectors, less than a batch
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                if (first + k * THREADS >= s.v1) break;
                sum.template add_vectors<T, 1>(raw + k, p.c);
            }
        }
    }
    const bool front = s.head && t < r.head, back = s.tail && r.tail() + t < p.classes;
    if (front) sum.add_one(to_f32<T>(gld(r.x + t)), Word<T>::low, p.c);
    if (back) sum.add_one(to_f32<T>(gld(r.x + r.tail() + t)), Word<T>::low, p.c);
    const uint32_t largest = s.v0 + t < s.v1 || front || back ? order_of(sum.m) : 0;
    auto join_all = [&](Part part) {
        part = join_block<THREADS>(part, parts, p.c);
        if constexpr (CLUSTER) {
            auto cluster = cg::this_cluster();
            if (t == 0) shared_part = part;
            cluster.sync();
            part = *cluster.map_shared_rank(&shared_part, 0);
            for (int b = 1; b < ranks; ++b) part = join(part, *cluster.map_shared_rank(&shared_part, b), p.c);
            cluster.sync();                            // nobody writes shared_part, or leaves, before all have read
        }
        return part;
    };
    Part all = join_all(sum.part());
    const float m = all.m == -INFINITY ? 0.0f : all.m;
    float l2s;
    if ((fabsf(m) > p.far && m < INFINITY) || m < Word<T>::lowest || p.careful) {                 // the whole row again, from its maximum
        Part again{0.0f, 0.0f, 0.0f};                  // (one origin for all: the sums add up)
        auto careful = [&](float x) {
            const float d = distance(x, m, p.c), e = exp2_fast(d);
            again.s += e;
            again.u = fmaf(e, d, again.u);
        };
        for (int v = s.v0 + t; v < s.v1; v += THREADS) {
            float x[VEC];
            unpack<T, VEC>(gldv<Raw<T, VEC>>(r.x + r.element(v)), x);
#pragma unroll
            for (int j = 0; j < VEC; ++j) careful(x[j]);
        }
        if (front) careful(to_f32<T>(gld(r.x + t)));
        if (back) careful(to_f32<T>(gld(r.x + r.tail() + t)));
        all = join_all(again);
        l2s = log2f(all.s);
    } else {
        l2s = log2f(all.s) - fmaf(m, p.c, -__fmul_rn(m, p.c));                // S from the exact product m * c
    }
    const RowResult result{m, all.s, all.u / all.s, l2s};
    if (t == 0 && rank == 0) store_row<T>(p, row, target, r.x, result, log2f(all.s));
    if constexpr (TOP) {
        const int top = p.top;
        block_top<T, THREADS>(sh, s, largest, top);
        if constexpr (CLUSTER) {
            auto cluster = cg::this_cluster();
            cluster.sync();
            if (rank == 0) {                           // the blocks' lists, each in order, ranked against one another
                for (int i = t; i < ranks * top; i += THREADS) lists[i] = cluster.map_shared_rank(sh.list, i / top)[i % top];
                __syncthreads();
                for (int i = t; i < ranks * top; i += THREADS) {
                    const unsigned long long k = lists[i];
                    int place = i % top;
                    for (int b = 0; b < ranks; ++b)
                        if (b != i / top) place += larger_than(lists + b * top, top, k);
                    if (k != 0 && place < top) store_top(p, row, place, k, result);
                }
            }
            cluster.sync();
        } else {
            if (t < top) store_top(p, row, t, sh.list[t], result);
        }
    }
}

constexpr int kShortThreads = 128;
// Rows of up to 8 * NB vectors, without alternatives: eight lanes each, the row in registers.  Joining a row's lanes and
// writing its results costs more instructions than so short a row itself; four rows of a warp share them.  65536 x 80 fp32:
// 7.7 us, by a warp for each row 18.6 (L2 holds the rows; 3.2 at the copy rate); 65536 x 256 bf16: 10.9 and 21.3.
constexpr int kPackedLanes = 8;
template <typename T, int NB>
__global__ void __launch_bounds__(kShortThreads)
log_probs_packed_kernel(const ProbsParams p)
{
    constexpr int VEC = RowView<T>::VEC, LANES = kPackedLanes, NS = (2 * (VEC - 1) + LANES - 1) / LANES;
    const int lane = threadIdx.x % LANES;
    const long long row = (long long)blockIdx.x * (kShortThreads / LANES) + threadIdx.x / LANES;
    const long long read = min(row, p.rows - 1);           // lanes behind the last row take part in the shuffles, and write nothing
    const RowView<T> r(static_cast<const T*>(p.x) + row_offset<unsigned>(read, p.inner, p.outer_stride, p.row_stride), p.classes);
    Raw<T, VEC> raw[NB];
#pragma unroll
    for (int k = 0; k < NB; ++k)
        if (lane + LANES * k < r.nvec) raw[k] = gldv<Raw<T, VEC>>(r.x + r.element(lane + LANES * k));
    float x[NB][VEC], x1[NS], m = -INFINITY;
#pragma unroll
    for (int k = 0; k < NS; ++k) {                         // the single elements in front and behind
        const int i = lane + LANES * k, one = i < r.head ? i : r.tail() + i - r.head;
        x1[k] = one < p.classes ? to_f32<T>(gld(r.x + one)) : -INFINITY;
        m = max_nan(m, x1[k]);
    }
    const long long target = p.target ? target_of(p.target, p.target64, read) : 0;
#pragma unroll
    for (int k = 0; k < NB; ++k) {
        unpack<T, VEC>(raw[k], x[k]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            if (lane + LANES * k >= r.nvec) x[k][j] = -INFINITY;
            m = max_nan(m, x[k][j]);
        }
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (m == -INFINITY) m = 0.0f;
    float s = 0.0f, u = 0.0f;
    auto add = [&](float v) {
        const float d = distance(v, m, p.c), e = exp2_fast(d);
        s += e;
        u = fmaf(e, d, u);
    };
#pragma unroll
    for (int k = 0; k < NS; ++k) add(x1[k]);
#pragma unroll
    for (int k = 0; k < NB; ++k)
#pragma unroll
        for (int j = 0; j < VEC; ++j) add(x[k][j]);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        u += __shfl_xor_sync(0xffffffffu, u, o);
    }
    if (lane != 0 || row >= p.rows) return;
    const float l2s = log2f(s);
    if (target < 0) store_unused(p, row, 0);
    else store_row<T>(p, row, target, r.x, {m, s, u / s, l2s}, l2s);
}

// Rows of up to 32 * NB vectors: a warp each, the row in registers.  The maximum is known before the sums are formed.
// 16384 x 1024 bf16: 10.6 us (L2 holds them); 65536 x 80 fp32 with 8 alternatives: 42 us, bound by the instructions that find
// them.
constexpr int kShortCandidates = 128;
template <typename T, int NB, bool TOP>
__global__ void __launch_bounds__(kShortThreads)
log_probs_short_kernel(const ProbsParams p)
{
    constexpr int VEC = RowView<T>::VEC, WARPS = kShortThreads / 32;
    __shared__ std::conditional_t<TOP, unsigned long long[WARPS][kShortCandidates], NoTop> candidates;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long row = (long long)blockIdx.x * WARPS + warp;
    if (row >= p.rows) return;
    const RowView<T> r(static_cast<const T*>(p.x) + row_offset<unsigned>(row, p.inner, p.outer_stride, p.row_stride), p.classes);
    // what a lane takes of the row: NB vectors, and one of the single elements in front and behind (at most 2 * (VEC - 1))
    Raw<T, VEC> raw[NB];
#pragma unroll
    for (int k = 0; k < NB; ++k)
        if (lane + 32 * k < r.nvec) raw[k] = gldv<Raw<T, VEC>>(r.x + r.element(lane + 32 * k));
    const int one = lane < r.head ? lane : r.tail() + lane - r.head;
    const bool single = one < p.classes;
    const float x1 = single ? to_f32<T>(gld(r.x + one)) : -INFINITY;
    const long long target = p.target ? target_of(p.target, p.target64, row) : 0;
    if (target < 0) {
        store_unused(p, row, lane);
        return;
    }
    float x[NB][VEC];
#pragma unroll
    for (int k = 0; k < NB; ++k) {
        unpack<T, VEC>(raw[k], x[k]);
        if (lane + 32 * k >= r.nvec) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) x[k][j] = -INFINITY;
        }
    }
    float mine = x1;
#pragma unroll
    for (int k = 0; k < NB; ++k)
#pragma unroll
        for (int j = 0; j < VEC; ++j) mine = max_nan(mine, x[k][j]);
    const float most = warp_max(mine), m = most == -INFINITY ? 0.0f : most;
    float s = 0.0f, u = 0.0f;
    auto add = [&](float v) {
        const float d = distance(v, m, p.c), e = exp2_fast(d);
        s += e;
        u = fmaf(e, d, u);
    };
    add(x1);
#pragma unroll
    for (int k = 0; k < NB; ++k)
#pragma unroll
        for (int j = 0; j < VEC; ++j) add(x[k][j]);
    warp_sum(s, u);
    const float l2s = log2f(s);
    const RowResult result{m, s, u / s, l2s};
    if (lane == 0) store_row<T>(p, row, target, r.x, result, l2s);
    if constexpr (TOP) {
        const int top = p.top;
        unsigned long long* cand = candidates[warp];
        // visit(key, whether it is one) by all lanes together
        auto visit = [&](auto&& f) {
#pragma unroll
            for (int k = 0; k < NB; ++k)
#pragma unroll
                for (int j = 0; j < VEC; ++j) f(x[k][j], r.element(lane + 32 * k) + j, lane + 32 * k < r.nvec);
            f(x1, one, single);
        };
        const uint32_t least = __shfl_sync(0xffffffffu, sort_descending(lane < r.nvec || single ? order_of(mine) : 0), top - 1);
        int n = 0;
        __syncwarp();
        visit([&](float v, int i, bool there) {
            const bool is = there && order_of(v) >= least;
            const unsigned ballot = __ballot_sync(0xffffffffu, is);
            const int at = n + __popc(ballot & ((1u << lane) - 1));
            if (is && at < kShortCandidates) cand[at] = key_of(v, i);
            n += __popc(ballot);
        });
        __syncwarp();
        if (n <= kShortCandidates) {
            for (int i = lane; i < n; i += 32) {
                const unsigned long long key = cand[i];
                int place = 0;
                for (int j = 0; j < n; ++j) place += cand[j] > key;
                if (place < top) store_top(p, row, place, key, result);
            }
        } else {                                       // more ties than the list holds: one after the other
            unsigned long long last = ~0ull;
            for (int place = 0; place < top; ++place) {
                unsigned long long key = 0;
                visit([&](float v, int i, bool there) {
                    const unsigned long long k = key_of(v, i);
                    if (there && k < last && k > key) key = k;
                });
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, o);
                    key = other > key ? other : key;
                }
                last = key;
                if (lane == 0) store_top(p, row, place, last, result);
            }
        }
        __syncwarp();
    }
}

// ---------------------------------------------------------------- backward
// TPR threads take kBatch vectors each of one row; `chunks` of them cover a row.  The last rows come first: they are
// what the forward pass has left in L2.  Vectors where x and dx have the same distance from a 16-byte boundary, else
// single elements.  ENTROPY: there is a gradient of the entropy (and 0 * -inf to be kept out).  4096 x 32768 bf16: 82 us, the
// copy rate, with issue slots 0.82 full.
constexpr int kBackThreads = 256;
template <typename T, int TPR, bool ENTROPY>
__global__ void __launch_bounds__(kBackThreads)
log_probs_backward_kernel(const ProbsBackParams p)
{
    constexpr int VEC = RowView<T>::VEC;
    using Index = std::conditional_t<TPR == kBackThreads, long long, unsigned>;
    const int t = threadIdx.x % TPR;
    const unsigned part = blockIdx.x * (kBackThreads / TPR) + threadIdx.x / TPR;   // (at most 2^31 + 8)
    const unsigned behind = part / (unsigned)p.chunks;
    const int chunk = (int)(part - behind * (unsigned)p.chunks);
    const long long row = p.rows - 1 - behind;
    if (row < 0) return;
    const T* x = static_cast<const T*>(p.x) + row_offset<Index>(row, p.inner, p.outer_stride, p.row_stride);
    T* dx = static_cast<T*>(p.dx) + row_offset<Index>(row, p.inner, p.dx_outer_stride, p.dx_row_stride);
    const RowView<T> r(x, p.classes);
    const bool same = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15) == 0;
    const int first = chunk * TPR * kBatch + t;
    Raw<T, VEC> raw[kBatch];
    if (same) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
            if (first + k * TPR < r.nvec) raw[k] = gldv<Raw<T, VEC>>(x + r.element(first + k * TPR));
    }
    const long long target = p.target ? target_of(p.target, p.target64, row) : 0;
    const float o = gld(p.stats + 3 * row), l2s = gld(p.stats + 3 * row + 1);
    const bool used = target >= 0 && l2s != -INFINITY;
    float g = 0.0f, gh = 0.0f, entropy = 0.0f;
    if (p.dlogp) g = target < p.classes ? gld(p.dlogp + row) : __int_as_float(0x7fffffff);
    if constexpr (ENTROPY) {
        gh = gld(p.dentropy + row);
        entropy = gld(p.stats + 3 * row + 2);
    }
    // dx = 2^d (a + b d), and g / T more at the target
    const float inv_s = exp2f(-l2s) * p.inv_temperature;
    const float a = -(g + gh * (entropy - kLn2 * l2s)) * inv_s, b = -gh * kLn2 * inv_s, at_target = g * p.inv_temperature;
    const int hot = p.dlogp && target < p.classes ? (int)target : -1;
    auto single = [&](int i) {
        float f = 0.0f;
        if (used) {
            const float d = distance(to_f32<T>(gld(x + i)), o, p.c);
            f = exp2_fast(d) * fmaf(b, d, a);
            if (i == hot) f += at_target;
        }
        gst(dx + i, from_f32<T>(f));
    };
    if (!same) {
        const int end = chunk == p.chunks - 1 ? p.classes : (chunk + 1) * TPR * kBatch * VEC;
        for (int i = chunk * TPR * kBatch * VEC + t; i < end; i += TPR) single(i);
        return;
    }
    const unsigned long long a2 = pair(a, a), b2 = pair(b, b), c2 = pair(p.c, p.c), o2 = pair(-o, -o);
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
        if (first + k * TPR < r.nvec) {
            const int i = r.element(first + k * TPR);
            float f[VEC];
            if (used) {
                unpack<T, VEC>(raw[k], f);
#pragma unroll
                for (int j = 0; j < VEC; j += 2) {
                    unsigned long long d = mul2(add2(pair(f[j], f[j + 1]), o2), c2), factor = a2;
                    unpair(d, f[j], f[j + 1]);
                    if constexpr (ENTROPY) {
                        f[j] = max_nan(f[j], kNoProbability);
                        f[j + 1] = max_nan(f[j + 1], kNoProbability);
                        factor = fma2(pair(f[j], f[j + 1]), b2, a2);
                    }
                    unpair(mul2(pair(exp2_fast(f[j]), exp2_fast(f[j + 1])), factor), f[j], f[j + 1]);
                }
                const unsigned at = (unsigned)(hot - i);
                if (at < (unsigned)VEC) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j)
                        if (at == (unsigned)j) f[j] += at_target;
                }
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) f[j] = 0.0f;
            }
            gstv(dx + i, pack<T, VEC>(f));
        }
    }
    if (chunk == 0 && t < r.head) single(t);
    if (chunk == p.chunks - 1 && r.tail() + t < p.classes) single(r.tail() + t);
}

// ---------------------------------------------------------------- host
template <typename T, int THREADS, bool TOP, bool CLUSTER>
int launch_with(cudaStream_t s, const ProbsParams& p, unsigned grid)
{
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(THREADS);
    cfg.stream = s;
    cudaLaunchAttribute attr{};
    if (CLUSTER) {
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = (unsigned)p.cluster;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
    }
    PXE_CUDA_OK(cudaLaunchKernelEx(&cfg, log_probs_kernel<T, THREADS, TOP, CLUSTER>, p));
    return PXE_OK;
}

template <typename T, int NB>
int launch_packed(cudaStream_t s, const ProbsParams& p)
{
    constexpr int rows = kShortThreads / kPackedLanes;
    log_probs_packed_kernel<T, NB><<<(unsigned)((p.rows + rows - 1) / rows), kShortThreads, 0, s>>>(p);
    PXE_LAUNCH_OK("log_probs_packed_kernel");
    return PXE_OK;
}

template <typename T, int NB, bool TOP>
int launch_short(cudaStream_t s, const ProbsParams& p)
{
    log_probs_short_kernel<T, NB, TOP><<<(unsigned)((p.rows + 3) / 4), kShortThreads, 0, s>>>(p);
    PXE_LAUNCH_OK("log_probs_short_kernel");
    return PXE_OK;
}

// A row to eight lanes up to 32 vectors without alternatives; to a warp, in its registers, up to 128 vectors, and without
// alternatives or in 32 bits up to 256 (16384 x 2000 bf16:
// 16 us, by blocks of 64 threads 24; its 8 alternatives take a warp 111 us and blocks of 128 threads 53).  Above, what a
// row's joining costs wants few threads where many rows wait, and few rows want many: up to 2048 vectors and when blocks
// of 256 threads could not hold all rows at once, 64 threads, or 128 that look for alternatives (16384 x 4000 bf16: 34 us
// against 61 by 256 threads, with alternatives 63 against 96; 8192 x 12001: 40 against 49; 4096 x 32768: 51 against 49).
// A cluster for rows of more than 4096 vectors, while all its blocks find room at once and every thread keeps a batch of
// vectors (1 x 131072 fp32: 6.4 us against 16.4, 16 x 128000 bf16: 6.6 against 12.6; 1 x 32000 bf16 with alternatives: 11.2
// in a cluster of eight against 7.8).
template <typename T>
int launch_forward(cudaStream_t s, ProbsParams& p, const DeviceInfo& di)
{
    const int vecs = p.classes / (16 / (int)sizeof(T));
    p.cluster = 1;
    if (p.top) {
        if (vecs <= 32) return launch_short<T, 1, true>(s, p);
        if (vecs <= 64) return launch_short<T, 2, true>(s, p);
        if (vecs <= 128) return launch_short<T, 4, true>(s, p);
        if constexpr (sizeof(T) == 4) { if (vecs <= 256) return launch_short<T, 8, true>(s, p); }
    } else {
        if (vecs <= kPackedLanes) return launch_packed<T, 1>(s, p);
        if (vecs <= 2 * kPackedLanes) return launch_packed<T, 2>(s, p);
        if (vecs <= 4 * kPackedLanes) return launch_packed<T, 4>(s, p);
        if (vecs <= 64) return launch_short<T, 2, false>(s, p);
        if (vecs <= 128) return launch_short<T, 4, false>(s, p);
        if (vecs <= 256) return launch_short<T, 8, false>(s, p);
    }
    if (vecs <= 2048 && p.rows > (long long)di.sm_count * kBlocks)
        return p.top ? launch_with<T, 128, true, false>(s, p, (unsigned)p.rows) : launch_with<T, 64, false, false>(s, p, (unsigned)p.rows);
    while (vecs > 4096 && p.cluster < 8 && p.rows * p.cluster * 2 <= 2LL * di.sm_count && vecs >= p.cluster * 2 * 256 * kBatch) p.cluster *= 2;
    const unsigned grid = (unsigned)(p.rows * p.cluster);
    if (p.cluster > 1) return p.top ? launch_with<T, 256, true, true>(s, p, grid) : launch_with<T, 256, false, true>(s, p, grid);
    return p.top ? launch_with<T, 256, true, false>(s, p, grid) : launch_with<T, 256, false, false>(s, p, grid);
}

// Eight lanes for rows of up to 32 vectors, a warp for every 128 vectors of rows of up to 512, a block for every 1024 of
// longer ones (65536 x 80 fp32: 7.5 us, by warps 23; 16384 x 4000 bf16: 51 by warps, 57 by blocks; 8192 x 8000: 50 by warps,
// 43 by blocks).
template <typename T, int TPR>
int launch_backward(cudaStream_t s, ProbsBackParams& p, int vecs)
{
    p.chunks = std::max(1, (vecs + TPR * kBatch - 1) / (TPR * kBatch));
    const long long rows = kBackThreads / TPR, blocks = (p.rows * p.chunks + rows - 1) / rows;
    PXE_REQUIRE(p.rows * p.chunks <= 0x80000000LL, "log_probs_backward: too many rows");
    auto kernel = p.dentropy ? log_probs_backward_kernel<T, TPR, true> : log_probs_backward_kernel<T, TPR, false>;
    kernel<<<(unsigned)blocks, kBackThreads, 0, s>>>(p);
    PXE_LAUNCH_OK("log_probs_backward_kernel");
    return PXE_OK;
}
template <typename T>
int launch_backward(cudaStream_t s, ProbsBackParams& p)
{
    const int vecs = p.classes / (16 / (int)sizeof(T));
    if (vecs <= 32) return launch_backward<T, 8>(s, p, vecs);
    return vecs <= 512 ? launch_backward<T, 32>(s, p, vecs) : launch_backward<T, kBackThreads>(s, p, vecs);
}

// Rows of x or dx: the checked strides; what the strides of a single row or a single group say is put aside.
int check_rows(const char* name, const void* ptr, int size, long long rows, long long& inner, long long& outer, long long& stride, int classes)
{
    PXE_REQUIRE(reinterpret_cast<uintptr_t>(ptr) % size == 0, "%s is not aligned to its elements", name);
    if (inner == 0) { inner = rows; outer = 0; }
    if (stride == 0) stride = classes;
    PXE_REQUIRE(inner > 0 && rows % inner == 0, "%s: %lld rows in groups of %lld", name, rows, inner);
    PXE_REQUIRE(stride >= classes, "%s: row stride %lld is less than %d classes", name, stride, classes);
    if (rows == inner) outer = 0;
    if (rows == 1) stride = classes;
    const long long covered = (inner - 1) * stride + classes;
    PXE_REQUIRE(rows == inner || outer >= covered, "%s: outer stride %lld, a group covers %lld", name, outer, covered);
    return PXE_OK;
}
// What such a tensor covers, in two ways that each cover all of it: its groups, and (where a group is a whole number of rows
// further) its rows.
struct Cover {
    RowSpan groups, rows;
};
Cover cover(const void* ptr, int size, long long rows, long long inner, long long outer, long long stride, int classes)
{
    const RowSpan groups{ptr, rows / inner, outer * size, ((inner - 1) * stride + classes) * size};
    if (rows != inner && outer % stride != 0) return {groups, groups};
    const long long lines = (rows / inner - 1) * (outer / stride) + inner;
    return {groups, {ptr, lines, stride * size, (long long)classes * size}};
}
bool conflict(const RowSpan& a, const Cover& b) { return rows_conflict(a, b.groups) && rows_conflict(a, b.rows); }
bool conflict(const Cover& a, const Cover& b)
{
    return rows_conflict(a.groups, b.groups) && rows_conflict(a.rows, b.rows) && rows_conflict(a.groups, b.rows) && rows_conflict(a.rows, b.groups);
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
    PXE_REQUIRE(d.temperature >= 1e-30f && d.temperature <= 1e30f, "log_probs: temperature %g is not in 1e-30..1e30", d.temperature);
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
    const Cover x = cover(d.x, size, d.rows, p.inner, p.outer_stride, p.row_stride, d.classes);
    const struct { const void* ptr; long long bytes; } outs[] = {{d.logp, d.rows * 4}, {d.entropy, d.rows * 4}, {d.stats, d.rows * 12},
                                                                 {d.top_logp, d.rows * d.top * 4}, {d.top_index, d.rows * d.top * 4}};
    PXE_REQUIRE(reinterpret_cast<uintptr_t>(d.target) % (d.target_is_int64 ? 8 : 4) == 0, "log_probs: target is not aligned to its elements");
    const RowSpan target{d.target, 1, 0, d.rows * (d.target_is_int64 ? 8 : 4)};
    for (const auto& o : outs) {
        if (!o.ptr) continue;
        const RowSpan span{o.ptr, 1, 0, o.bytes};
        PXE_REQUIRE(reinterpret_cast<uintptr_t>(o.ptr) % 4 == 0, "log_probs: an output is not aligned to its elements");
        PXE_REQUIRE(o.ptr != d.x && o.ptr != d.target && !conflict(span, x) && !rows_conflict(span, target), "log_probs: an output overlaps an input");
        for (const auto& other : outs)
            PXE_REQUIRE(&other == &o || !other.ptr || (other.ptr != o.ptr && !rows_conflict(span, {other.ptr, 1, 0, other.bytes})),
                        "log_probs: two outputs overlap");
    }
    DeviceInfo di;
    { const int rc = device_info(&di); if (rc != PXE_OK) return rc; }
    p.careful = !(p.c > 0.02f && p.c < 1e7f);              // what -inf is held at would count, or overflow
    p.far = kFar / p.c;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (d.type == PXE_F32) return launch_forward<float>(s, p, di);
    if (d.type == PXE_BF16) return launch_forward<bf16>(s, p, di);
    return launch_forward<f16>(s, p, di);
}

extern "C" int pxe_log_probs_backward(pxe_stream_t stream, const pxe_log_probs_backward_desc* dp)
{
    PXE_REQUIRE(dp != nullptr, "log_probs_backward: null descriptor");
    const pxe_log_probs_backward_desc& d = *dp;
    PXE_REQUIRE(valid_dtype(d.type), "log_probs_backward: unknown type %d", d.type);
    PXE_REQUIRE(d.rows >= 0 && d.classes > 0, "log_probs_backward: shape [%lld, %d]", d.rows, d.classes);
    PXE_REQUIRE(d.rows <= 0x7fffffffLL, "log_probs_backward: too many rows");
    PXE_REQUIRE(d.classes <= (1 << 30), "log_probs_backward: too many classes");
    PXE_REQUIRE(d.temperature >= 1e-30f && d.temperature <= 1e30f, "log_probs_backward: temperature %g is not in 1e-30..1e30", d.temperature);
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
    int rc = check_rows("log_probs_backward: x", d.x, size, d.rows, p.inner, p.outer_stride, p.row_stride, d.classes);
    if (rc == PXE_OK) rc = check_rows("log_probs_backward: dx", d.dx, size, d.rows, inner, p.dx_outer_stride, p.dx_row_stride, d.classes);
    if (rc != PXE_OK) return rc;
    const Cover x = cover(d.x, size, d.rows, p.inner, p.outer_stride, p.row_stride, d.classes);
    const Cover dx = cover(d.dx, size, d.rows, inner, p.dx_outer_stride, p.dx_row_stride, d.classes);
    PXE_REQUIRE(d.dx == d.x ? p.row_stride == p.dx_row_stride && p.outer_stride == p.dx_outer_stride : !conflict(dx, x),
                "log_probs_backward: dx partially overlaps x");
    const int tsize = d.target_is_int64 ? 8 : 4;
    const struct { const void* ptr; long long bytes; int align; } ins[] = {{d.stats, d.rows * 12, 4}, {d.dlogp, d.rows * 4, 4},
                                                                           {d.dentropy, d.rows * 4, 4}, {d.target, d.rows * tsize, tsize}};
    for (const auto& i : ins) {
        PXE_REQUIRE(reinterpret_cast<uintptr_t>(i.ptr) % i.align == 0, "log_probs_backward: an input is not aligned to its elements");
        PXE_REQUIRE(!i.ptr || (i.ptr != d.dx && !conflict(RowSpan{i.ptr, 1, 0, i.bytes}, dx)), "log_probs_backward: dx overlaps an input");
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (d.type == PXE_F32) return launch_backward<float>(s, p);
    if (d.type == PXE_BF16) return launch_backward<bf16>(s, p);
    return launch_backward<f16>(s, p);
}
