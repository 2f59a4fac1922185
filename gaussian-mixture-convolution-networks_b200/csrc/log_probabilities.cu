// Log-probabilities of given classes, entropy and top alternatives of rows of logits, and their gradient.
//
//   x_j = z_j - max z,  s = sum_j e^(x_j / T),  log p_j = x_j / T - log s,  H = log s - (sum_j e^(x_j / T) x_j / T) / s
//   dz_j = 1/T [ g_t d(t, j) + sum_i g_i d(i-th alternative, j) - p_j (g_t + sum_i g_i) - p_j g_H (log p_j + H) ]
//
// Every sum is held in fp32 relative to the running maximum (m, s, t = sum e x), so a row is read once whatever its
// length. Masked classes (-inf, or the type's lowest value) need no branch: e = 0 there and x is bounded from below
// before it is multiplied by e. A row with nothing but -inf has no distribution: log p = -inf, H = 0, gradient 0.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace gmc {
namespace {

namespace cg = cooperative_groups;
typedef unsigned long long Key;

constexpr int kMaxTop = 32;              // a warp keeps a sorted list of alternatives, one per lane
constexpr int kRowThreads = 256;         // long rows: threads of a CTA
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kUnroll = 4;               // 16-byte vectors a thread has in flight
constexpr int kSmallThreads = 128;       // short rows: one warp per row, four rows per CTA
constexpr int kSmallClasses = 1024;      // at most 32 elements per lane
constexpr float kLowest = -1e20f;        // bound of x: e is 0 far above it for every temperature allowed, 0 * kLowest = -0
constexpr float kNearLowest = -1e35f;    // z above it: z minus any finite 16-bit maximum stays in the fp32 range
constexpr float kMinTemperature = 1e-6f, kMaxTemperature = 1e6f;

__device__ __forceinline__ float neg_inf() { return __int_as_float(0xff800000); }
__device__ __forceinline__ float quiet_nan() { return __int_as_float(0x7fffffff); }

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// 16 bytes of a row as floats.
template <typename T>
struct Vec {
    static constexpr int N = 16 / int(sizeof(T));
    union { uint4 raw; T e[N]; };
    __device__ __forceinline__ float at(int i) const { return to_float<T>(e[i]); }
};
template <>
__device__ __forceinline__ float Vec<__nv_bfloat16>::at(int i) const {
    const unsigned w = i < 2 ? raw.x : i < 4 ? raw.y : i < 6 ? raw.z : raw.w;
    return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
}
template <typename T> __device__ __forceinline__ uint4 masked_vector();          // a vector of -inf
template <> __device__ __forceinline__ uint4 masked_vector<float>() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
template <> __device__ __forceinline__ uint4 masked_vector<__nv_bfloat16>() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
template <> __device__ __forceinline__ uint4 masked_vector<__half>() { return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u); }

// Largest and smallest of a thread's vectors, NaN left out. 16-bit types are compared in pairs.
template <typename T>
__device__ __forceinline__ void extremes(const Vec<T> (&v)[kUnroll], float& largest, float& smallest) {
    if constexpr (sizeof(T) == 2) {
        using Pair = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
        Pair hi, lo;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const Pair* p = reinterpret_cast<const Pair*>(&v[u].raw);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                hi = u + i == 0 ? p[0] : __hmax2(hi, p[i]);
                lo = u + i == 0 ? p[0] : __hmin2(lo, p[i]);
            }
        }
        largest = fmaxf(to_float<T>(hi.x), to_float<T>(hi.y));
        smallest = fminf(to_float<T>(lo.x), to_float<T>(lo.y));
    } else {
        largest = v[0].at(0);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
#pragma unroll
            for (int i = 0; i < Vec<T>::N; ++i) largest = fmaxf(largest, v[u].at(i));
        smallest = neg_inf();                                                       // comparing again would cost what the bound costs
    }
}

// Order of the alternatives as one number: larger value first, then lower index. NaN ranks behind -inf; 0 is no element.
__device__ __forceinline__ Key make_key(float z, unsigned index) {
    const int b = __float_as_int(z + 0.f);                                         // -0 and +0 are equal
    const unsigned order = z != z ? 1u : (b >= 0 ? unsigned(b) | 0x80000000u : ~unsigned(b));
    return (Key(order) << 32) | (0xffffffffu - index);
}
__device__ __forceinline__ unsigned key_index(Key k) { return 0xffffffffu - unsigned(k); }
__device__ __forceinline__ float key_value(Key k) {
    const unsigned order = unsigned(k >> 32);
    return order == 1u ? quiet_nan() : __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
__device__ __forceinline__ Key warp_max(Key k) {
    const unsigned hi = __reduce_max_sync(0xffffffffu, unsigned(k >> 32));
    const unsigned lo = __reduce_max_sync(0xffffffffu, unsigned(k >> 32) == hi ? unsigned(k) : 0u);
    return (Key(hi) << 32) | lo;
}

// Running maximum m, s = sum e^((z - m) / T) and t = sum e^((z - m) / T) (z - m); k = log2(e) / T.
struct Stat {
    float m, s, t;
};
__device__ __forceinline__ void raise(Stat& a, float m, float k) {
    if (a.s > 0.f) {
        const float d = fmaxf(a.m - m, kLowest);
        const float f = ex2_approx(d * k);
        a.t = f * (a.t + d * a.s);
        a.s *= f;
    }
    a.m = m;
}
// Over the lanes: the maximum first, then one rescaling and two sums (a merge of pairs would rescale in each of five steps).
__device__ __forceinline__ Stat warp_merge(Stat a, float k) {
    float m = a.m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    raise(a, m, k);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
        a.t += __shfl_xor_sync(0xffffffffu, a.t, o);
    }
    return a;
}
// e^(x / T) by the approximate base-2 exponential (error 2^-22 of itself) of x k rounded to fp32, 2^-24 |x k|: terms that count have
// |x k| of a few, up to log2 of the row's length, and log p comes out to 1e-7, as with expf of a rounded x / T (1 x 50257:
// 1.0e-7 against 0.6e-7 of plain fp32 operations, 5e-7 seen); one multiplication and one special-function instruction a term.
__device__ __forceinline__ void add_element(float z, float base, float k, float& s, float& t) {
    const float x = z - base;
    const float e = ex2_approx(x * k);
    s += e;
    t += e * fmaxf(x, kLowest);
}

// Two elements at once: packed additions and products take one issue slot for both. BOUND: x may be -inf.
template <bool BOUND>
__device__ __forceinline__ void add_pair(float2 z, float2 minus_base, float2 k, float2& s, float2& t) {
    const float2 x = __fadd2_rn(z, minus_base), y = __fmul2_rn(x, k);
    const float2 e = make_float2(ex2_approx(y.x), ex2_approx(y.y));
    s = __fadd2_rn(s, e);
    t = __ffma2_rn(e, BOUND ? make_float2(fmaxf(x.x, kLowest), fmaxf(x.y, kLowest)) : x, t);
}
template <bool BOUND, typename T>
__device__ __forceinline__ void add_vectors(const Vec<T> (&v)[kUnroll], float base, float k, Stat& st) {
    float2 s = make_float2(0.f, 0.f), t = s;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
        for (int i = 0; i < Vec<T>::N; i += 2)
            add_pair<BOUND>(make_float2(v[u].at(i), v[u].at(i + 1)), make_float2(-base, -base), make_float2(k, k), s, t);
    st.s += s.x + s.y;
    st.t += t.x + t.y;
}

// (z - m) / T: the difference of two finite logits may leave the fp32 range where the quotient does not.
__device__ __forceinline__ float scaled(float z, float m, float inv_t) {
    const float x = z - m;
    return x == neg_inf() && z != neg_inf() ? z * inv_t - m * inv_t : x * inv_t;
}

struct Outputs {
    float* target;                // [n_rows] or null
    float* entropy;               // [n_rows]
    float* stats;                 // [n_rows, 2]: maximum and log s, for the gradient; or null
    float* top;                   // [n_rows, n_top]
    long long* top_indices;
};

// The target of a row and its logit, read early: the outputs come at the end of a chain of latencies.
struct Target {
    long long t;
    float z;
};
template <typename T>
__device__ __forceinline__ Target read_target(const T* z, const long long* targets, long long row, int n_classes, long long ignored) {
    Target g = {ignored, 0.f};
    if (targets) {
        g.t = targets[row];
        if (g.t >= 0 && g.t < n_classes) g.z = to_float<T>(z[g.t]);
    }
    return g;
}
// One thread: the row's outputs apart from the alternatives. Returns log s.
__device__ __forceinline__ float write_row(const Outputs& out, const Stat& st, const Target& g, long long row, int n_classes, long long ignored,
                                           float inv_t) {
    const bool empty = st.m == neg_inf() && st.s == 0.f;
    const float log_s = logf(st.s);
    out.entropy[row] = empty ? 0.f : log_s - inv_t * (st.t / st.s);
    if (out.stats) {
        out.stats[2 * row] = st.m;
        out.stats[2 * row + 1] = log_s;
    }
    if (out.target) {
        float v;
        if (g.t == ignored) {
            v = 0.f;
        } else if (g.t < 0 || g.t >= n_classes) {
            report_check(CHECK_CLASS_RANGE);
            v = quiet_nan();
        } else {
            v = empty ? neg_inf() : scaled(g.z, st.m, inv_t) - log_s;
        }
        out.target[row] = v;
    }
    return log_s;
}
__device__ __forceinline__ void write_alternative(const Outputs& out, Key key, long long row, int n_top, int place, float m, float log_s,
                                                  bool empty, float inv_t) {
    out.top_indices[row * n_top + place] = (long long)key_index(key);
    out.top[row * n_top + place] = empty ? neg_inf() : scaled(key_value(key), m, inv_t) - log_s;
}

// ---- short rows: one warp per row, the row in registers ---------------------------------------------------------------
// At most 1024 classes. Bound by one chain of latencies (launch, load, two reductions over the warp, stores): 5.3 us for one row
// of 10 classes and for 256 rows of 40 with the caches cold, where the bytes alone would take 0.02 us. The alternatives are
// found by n_top maxima over the warp, each below the one before.
template <typename T, int E>
__global__ void __launch_bounds__(kSmallThreads) forward_small_kernel(const T* __restrict__ logits, const long long* __restrict__ targets,
                                                                      long long n_rows, int n_classes, long long row_stride,
                                                                      float inv_t, float k, long long ignored, int n_top, Outputs out) {
    const long long row = ((long long)blockIdx.x * kSmallThreads + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    if (row >= n_rows) return;
    const T* z = logits + row * row_stride;
    float v[E];
    Stat st = {neg_inf(), 0.f, 0.f};
    const Target given = lane == 0 ? read_target<T>(z, targets, row, n_classes, ignored) : Target{ignored, 0.f};
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int c = lane + 32 * i;
        v[i] = c < n_classes ? to_float<T>(z[c]) : neg_inf();
        st.m = fmaxf(st.m, v[i]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) st.m = fmaxf(st.m, __shfl_xor_sync(0xffffffffu, st.m, o));
    const float base = st.m == neg_inf() ? 0.f : st.m;
#pragma unroll
    for (int i = 0; i < E; ++i) add_element(v[i], base, k, st.s, st.t);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        st.s += __shfl_xor_sync(0xffffffffu, st.s, o);
        st.t += __shfl_xor_sync(0xffffffffu, st.t, o);
    }
    float log_s = 0.f;
    if (lane == 0) log_s = write_row(out, st, given, row, n_classes, ignored, inv_t);
    if (n_top == 0) return;
    log_s = __shfl_sync(0xffffffffu, log_s, 0);
    // the k-th alternative is the largest key below the one before it
    Key last = ~Key(0), mine = 0;
    for (int place = 0; place < n_top; ++place) {
        Key best = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int c = lane + 32 * i;
            const Key key = make_key(v[i], unsigned(c));
            if (c < n_classes && key < last && key > best) best = key;
        }
        last = warp_max(best);
        if (lane == place) mine = last;
    }
    if (lane < n_top) write_alternative(out, mine, row, n_top, lane, st.m, log_s, st.m == neg_inf() && st.s == 0.f, inv_t);
}

// ---- long rows: a CTA, or a cluster of up to eight, per row ----------------------------------------------------------
// The row is cut into single elements up to the first 16-byte boundary, whole vectors, and single elements behind the last
// one. The vectors are dealt to the CTAs of the cluster in contiguous parts; the single elements go to CTA 0.
template <typename T>
struct Row {
    const T* z;
    int head, n_vec, tail;         // elements, vectors, elements
    int first, end;                // vectors of this CTA
    bool singles;
    __device__ __forceinline__ Row(const T* row, int n_classes, int rank, int n_ranks) : z(row) {
        constexpr int N = Vec<T>::N;
        head = min(n_classes, int((16u - unsigned(reinterpret_cast<uintptr_t>(row) & 15u)) & 15u) / int(sizeof(T)));
        n_vec = (n_classes - head) / N;
        tail = n_classes - head - n_vec * N;
        first = int((long long)n_vec * rank / n_ranks);
        end = int((long long)n_vec * (rank + 1) / n_ranks);
        singles = rank == 0;
    }
    __device__ __forceinline__ int element(int vector) const { return head + vector * Vec<T>::N; }
    __device__ __forceinline__ Vec<T> load(int vector) const {
        Vec<T> v;
        v.raw = vector < end ? __ldg(reinterpret_cast<const uint4*>(z + element(vector))) : masked_vector<T>();
        return v;
    }
};

// Sorted list of the warp's largest keys, one per lane, descending; keys that arrive are all different.
__device__ __forceinline__ void list_insert(Key& list, Key key, int lane) {
    const int place = __popc(__ballot_sync(0xffffffffu, list > key));
    const Key above = __shfl_up_sync(0xffffffffu, list, 1);
    if (lane == place) list = key;
    else if (lane > place) list = above;
}
__device__ __forceinline__ void list_offer(Key& list, Key& bound, Key key, int n_top, int lane) {
    unsigned waiting = __ballot_sync(0xffffffffu, key > bound);
    while (waiting) {
        const int src = __ffs(waiting) - 1;
        list_insert(list, __shfl_sync(0xffffffffu, key, src), lane);
        const Key last = __shfl_sync(0xffffffffu, list, n_top - 1);
        bound = last > bound ? last : bound;
        waiting &= __ballot_sync(0xffffffffu, key > bound);
        waiting &= ~(1u << src);
    }
}
// Number of keys above `key` among n keys in shared memory, which are all different.
__device__ __forceinline__ int rank_among(const Key* keys, int n, Key key) {
    int rank = 0;
#pragma unroll 4
    for (int i = 0; i < n; ++i) rank += keys[i] > key ? 1 : 0;
    return rank;
}

// Alternatives without a second look at most of the row. After the sums every thread knows its largest element; the n_top-th
// largest of the 32 maxima of groups of eight threads is a value that at least n_top elements reach, and few more than that
// do (about 30 for 20 of independent values). The threads whose maximum reaches it read their elements again and collect
// those that do; a collected element's place is the number of larger ones (the order of the atomic additions that hand out the
// collecting places does not matter). Where too many are equal (a constant row), the
// warps go through all their elements and keep sorted lists instead.
//
// Many rows of 16-bit logits are bound by issue: 4093 x 32003 in bf16 57 us, 4.6 TB/s of the copy's 6.5, with 70 % of the issue
// slots and 61 % of the exponential unit in use. fp32 has half the classes per byte: 1021 x 100003 with four alternatives 76 us,
// 5.4 TB/s. Few rows are bound by latencies (launch of the cluster, first loads, three reductions, the alternatives): 64 rows of
// 131072 in bf16 with eight alternatives 16 us, 1 TB/s; one row of 50257 with 20 alternatives 15 us with the caches cold.
constexpr int kCollected = 512;
template <typename T, bool TOP>
__global__ void __launch_bounds__(kRowThreads, 4) forward_row_kernel(const T* __restrict__ logits, const long long* __restrict__ targets,
                                                                  int n_classes, long long row_stride, int n_ranks, float inv_t, float k,
                                                                  long long ignored, int n_top, Outputs out) {
    constexpr int N = Vec<T>::N;
    __shared__ Stat warp_stat[kRowWarps];
    __shared__ Stat cta_stat;
    __shared__ float group_max[32], row_log_s;
    __shared__ Key collected[kCollected];
    __shared__ Key cta_list[kMaxTop];
    __shared__ int count;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = int(blockIdx.x % unsigned(n_ranks));
    const long long row = blockIdx.x / unsigned(n_ranks);
    const Row<T> r(logits + row * row_stride, n_classes, rank, n_ranks);
    const Target given = tid == 0 && rank == 0 ? read_target<T>(r.z, targets, row, n_classes, ignored) : Target{ignored, 0.f};

    Stat st = {neg_inf(), 0.f, 0.f};
    const bool has_head = r.singles && tid < r.head, has_tail = r.singles && tid < r.tail;
    const int tail_first = r.head + r.n_vec * N;
    if (has_head) {
        const float z = to_float<T>(r.z[tid]);
        if (z > st.m) st.m = z;
        add_element(z, st.m == neg_inf() ? 0.f : st.m, k, st.s, st.t);
    }
    Vec<T> next[kUnroll];                                                           // on its way while the last ones are added up
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) next[u] = r.load(r.first + tid + u * kRowThreads);
    for (int of_warp = r.first + warp * 32; of_warp < r.end; of_warp += kRowThreads * kUnroll) {
        Vec<T> v[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            v[u] = next[u];
            next[u] = r.load(of_warp + lane + (kUnroll + u) * kRowThreads);
        }
        float m, least;
        extremes<T>(v, m, least);
        if (m > st.m) raise(st, m, k);
        const float base = st.m == neg_inf() ? 0.f : st.m;
        if (sizeof(T) == 2 && __all_sync(0xffffffffu, least > kNearLowest)) add_vectors<false, T>(v, base, k, st);
        else add_vectors<true, T>(v, base, k, st);
    }
    if (has_tail) {
        const float z = to_float<T>(r.z[tail_first + tid]);
        if (z > st.m) raise(st, z, k);
        add_element(z, st.m == neg_inf() ? 0.f : st.m, k, st.s, st.t);
    }

    const float mine = st.m;
    if constexpr (TOP) {
        float m = mine;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if ((lane & 7) == 0) group_max[tid >> 3] = m;
        if (tid == 0) count = 0;
        if (tid < kMaxTop) cta_list[tid] = 0;
    }
    st = warp_merge(st, k);
    if (lane == 0) warp_stat[warp] = st;
    __syncthreads();
    // all warps' sums, by the lanes of the first one
    if (warp == 0) {
        st = warp_merge(lane < kRowWarps ? warp_stat[lane] : Stat{neg_inf(), 0.f, 0.f}, k);
        if (lane == 0) {
            cta_stat = st;
            if (n_ranks == 1) row_log_s = write_row(out, st, given, row, n_classes, ignored, inv_t);
        }
    }
    if constexpr (TOP) {
        // every warp finds the n_top-th of the groups' maxima
        const float m = group_max[lane];
        int above = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const float other = __shfl_sync(0xffffffffu, m, i);
            above += other > m || (other == m && i < lane) ? 1 : 0;
        }
        const float bar = __shfl_sync(0xffffffffu, m, __ffs(__ballot_sync(0xffffffffu, above == n_top - 1)) - 1);
        auto collect = [&](float z, int c) {
            if (z >= bar) {
                const int place = atomicAdd(&count, 1);
                if (place < kCollected) collected[place] = make_key(z, unsigned(c));
            }
        };
        if (bar > neg_inf()) {
            if (has_head) collect(to_float<T>(r.z[tid]), tid);
            if (has_tail) collect(to_float<T>(r.z[tail_first + tid]), tail_first + tid);
            // a thread's vectors by its whole warp: one after the other they would each wait for the memory
            unsigned owners = __ballot_sync(0xffffffffu, mine >= bar);
            while (owners) {
                const int owner = (warp << 5) + __ffs(owners) - 1;
                owners &= owners - 1;
                for (int at0 = r.first + owner; at0 < r.end; at0 += kRowThreads * 32 * 2) {
                    Vec<T> v[2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) v[u] = r.load(at0 + (u * 32 + lane) * kRowThreads);
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int i = 0; i < N; ++i) collect(v[u].at(i), r.element(at0 + (u * 32 + lane) * kRowThreads) + i);
                }
            }
        }
        __syncthreads();
        int n = count;
        if (n > kCollected || bar == neg_inf()) {
            __syncthreads();                                                        // count and collected are replaced
            Key list = 0, bound = 0;
            if (r.singles) {
                list_offer(list, bound, has_head ? make_key(to_float<T>(r.z[tid]), unsigned(tid)) : 0, n_top, lane);
                list_offer(list, bound, has_tail ? make_key(to_float<T>(r.z[tail_first + tid]), unsigned(tail_first + tid)) : 0, n_top, lane);
            }
            for (int at0 = r.first + warp * 32; at0 < r.end; at0 += kRowThreads) {
                const int at = at0 + lane;
                const Vec<T> v = r.load(at);
#pragma unroll
                for (int i = 0; i < N; ++i)
                    list_offer(list, bound, at < r.end ? make_key(v.at(i), unsigned(r.element(at) + i)) : 0, n_top, lane);
            }
            collected[tid] = list;
            __syncthreads();
            n = kRowThreads;
        }
        for (int i = tid; i < n; i += kRowThreads) {
            const Key key = collected[i];
            const int place = key ? rank_among(collected, n, key) : kRowThreads;
            if (place < n_top) cta_list[place] = key;
        }
        __syncthreads();
    }
    if (n_ranks == 1) {
        if constexpr (TOP) {
            if (tid < n_top)
                write_alternative(out, cta_list[tid], row, n_top, tid, cta_stat.m, row_log_s, cta_stat.m == neg_inf() && cta_stat.s == 0.f, inv_t);
        }
        return;
    }
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (rank == 0) {
        const int total = n_ranks * n_top;
        if constexpr (TOP) {
            for (int i = tid; i < total; i += kRowThreads) collected[i] = cluster.map_shared_rank(cta_list, i / n_top)[i % n_top];
        }
        if (warp == 0) {
            st = warp_merge(lane < n_ranks ? *cluster.map_shared_rank(&cta_stat, lane) : Stat{neg_inf(), 0.f, 0.f}, k);
            if (lane == 0) {
                warp_stat[0] = st;
                row_log_s = write_row(out, st, given, row, n_classes, ignored, inv_t);
            }
        }
        if constexpr (TOP) {
            __syncthreads();
            const Stat all = warp_stat[0];
            for (int i = tid; i < total; i += kRowThreads) {
                const Key key = collected[i];
                const int place = key ? rank_among(collected, total, key) : kRowThreads;
                if (place < n_top) write_alternative(out, key, row, n_top, place, all.m, row_log_s, all.m == neg_inf() && all.s == 0.f, inv_t);
            }
        }
    }
    cluster.sync();                                                                 // shared memory is read by CTA 0 until here
}

// ---- gradient --------------------------------------------------------------------------------------------------------
struct Incoming {
    const float* target;            // [n_rows] each, [n_rows, n_top] for top; null = zero
    const float* entropy;
    const float* top;
};
struct RowGradient {                // grad_j = p_j (a + b x_j), x_j = z_j - m, plus the given classes' own terms
    float m, a, b, g_target, log2_s;
    float lowest;                   // bound of x_j far below where p_j is 0, for which b times it stays finite
    long long target;
    bool empty, bad;
};
__device__ __forceinline__ RowGradient row_gradient(const Incoming& in, const float* stats, const float* entropy, const long long* targets,
                                                    long long row, int n_classes, long long ignored, int n_top, float inv_t) {
    RowGradient g;
    g.m = stats[2 * row];
    const float log_s = stats[2 * row + 1], h = entropy[row];
    g.log2_s = log_s * kLog2e;
    g.empty = g.m == neg_inf() && log_s == neg_inf();
    g.target = in.target ? targets[row] : ignored;
    g.bad = g.target != ignored && (g.target < 0 || g.target >= n_classes);
    g.g_target = g.target != ignored && !g.bad ? in.target[row] : 0.f;
    float sum = g.g_target;
    if (in.top)
        for (int i = 0; i < n_top; ++i) sum += in.top[row * n_top + i];
    // -p_j / T (sum + g_H (x_j / T - log s + H))
    const float g_h = in.entropy ? in.entropy[row] : 0.f;
    g.a = -inv_t * (sum + g_h * (h - log_s));
    g.b = -inv_t * g_h * inv_t;
    g.lowest = -1000.f / inv_t;
    return g;
}
__device__ __forceinline__ float2 gradient_pair(const RowGradient& g, float2 z, float k) {
    const float2 x = __fadd2_rn(z, make_float2(-g.m, -g.m));
    const float2 y = __ffma2_rn(x, make_float2(k, k), make_float2(-g.log2_s, -g.log2_s));
    const float2 p = make_float2(ex2_approx(y.x), ex2_approx(y.y));
    return __fmul2_rn(p, __ffma2_rn(make_float2(fmaxf(x.x, g.lowest), fmaxf(x.y, g.lowest)), make_float2(g.b, g.b), make_float2(g.a, g.a)));
}
__device__ __forceinline__ float gradient_at(const RowGradient& g, float z, float k) { return gradient_pair(g, make_float2(z, z), k).x; }
// One thread: the whole gradient at the i-th given class (0 = the target, 1.. = the alternatives) of a row, written once
// for classes that are given more than once.
template <typename T>
__device__ __forceinline__ void given_class(const RowGradient& g, const Incoming& in, const long long* top_indices, const T* z, T* grad,
                                            long long row, int n_top, int i, int from, int to, float inv_t, float k) {
    const long long* tops = top_indices + row * n_top;
    const long long c = i == 0 ? (g.target >= 0 && g.g_target != 0.f ? g.target : -1) : tops[i - 1];
    if (c < from || c >= to) return;
    float own = i == 0 ? g.g_target : in.top[row * n_top + i - 1];
    if (i > 0 && c == g.target && g.g_target != 0.f) return;                        // written with the target
    if (i == 0 && in.top)
        for (int j = 0; j < n_top; ++j)
            if (tops[j] == c) own += in.top[row * n_top + j];
    grad[c] = from_float<T>(gradient_at(g, to_float<T>(z[c]), k) + own * inv_t);
}

template <typename T, int E>
__global__ void __launch_bounds__(kSmallThreads) backward_small_kernel(const T* __restrict__ logits, const long long* __restrict__ targets,
                                                                       const long long* __restrict__ top_indices,
                                                                       const float* __restrict__ stats, const float* __restrict__ entropy,
                                                                       Incoming in, T* __restrict__ grad, long long n_rows, int n_classes,
                                                                       long long row_stride, float inv_t, float k, long long ignored,
                                                                       int n_top) {
    const long long row = ((long long)blockIdx.x * kSmallThreads + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    if (row >= n_rows) return;
    const T* z = logits + row * row_stride;
    T* dz = grad + row * n_classes;
    const RowGradient g = row_gradient(in, stats, entropy, targets, row, n_classes, ignored, n_top, inv_t);
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int c = lane + 32 * i;
        if (c < n_classes) {
            const float v = gradient_at(g, to_float<T>(z[c]), k);
            dz[c] = from_float<T>(g.bad ? quiet_nan() : g.empty ? 0.f : v);
        }
    }
    if (g.bad || g.empty) return;
    __syncwarp();                                                                   // the warp's stores before the given classes'
    for (int i = lane; i < 1 + (in.top ? n_top : 0); i += 32)
        given_class<T>(g, in, top_indices, z, dz, row, n_top, i, 0, n_classes, inv_t, k);
}

// Long rows: a CTA per stretch of kStretch vectors of a row. Bound by the memory, one read and one write: 4093 x 32003 in bf16
// 91 us, 5.8 TB/s; 1021 x 100003 in fp32 135 us, 6.0 TB/s. Written past the caches (__stcs), which leaves the L2 cache to the
// rows that the forward pass has read last.
constexpr int kStretch = kRowThreads * kUnroll;
template <typename T>
__global__ void __launch_bounds__(kRowThreads) backward_row_kernel(const T* __restrict__ logits, const long long* __restrict__ targets,
                                                                   const long long* __restrict__ top_indices,
                                                                   const float* __restrict__ stats, const float* __restrict__ entropy,
                                                                   Incoming in, T* __restrict__ grad, int n_stretches, int n_classes,
                                                                   long long row_stride, float inv_t, float k, long long ignored, int n_top) {
    constexpr int N = Vec<T>::N;
    const int tid = threadIdx.x;
    // from the last row to the first: the forward pass has left the last ones in the L2 cache
    const unsigned cta = gridDim.x - 1 - blockIdx.x;
    const long long row = cta / unsigned(n_stretches);
    const int stretch = int(cta % unsigned(n_stretches));
    const T* z = logits + row * row_stride;
    T* dz = grad + row * n_classes;
    const bool vectors = ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(dz)) & 15u) == 0;
    Row<T> r(z, n_classes, 0, 1);
    r.first = min(stretch * kStretch, r.n_vec);
    r.end = min(r.n_vec, r.first + kStretch);
    Vec<T> v[kUnroll];
    if (vectors) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) v[u] = r.load(r.first + tid + u * kRowThreads);
    }
    const RowGradient g = row_gradient(in, stats, entropy, targets, row, n_classes, ignored, n_top, inv_t);
    const bool constant = g.bad || g.empty;
    const float value = g.bad ? quiet_nan() : 0.f;
    int from, to;                                                                   // elements of this CTA
    if (vectors) {
        from = stretch == 0 ? 0 : r.element(r.first);
        to = stretch == n_stretches - 1 ? n_classes : r.element(r.end);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int at = r.first + tid + u * kRowThreads;
            if (at < r.end) {
                Vec<T> w;
#pragma unroll
                for (int i = 0; i < N; i += 2) {
                    const float2 d = gradient_pair(g, make_float2(v[u].at(i), v[u].at(i + 1)), k);
                    w.e[i] = from_float<T>(constant ? value : d.x);
                    w.e[i + 1] = from_float<T>(constant ? value : d.y);
                }
                __stcs(reinterpret_cast<uint4*>(dz + r.element(at)), w.raw);
            }
        }
        if (stretch == 0 && tid < r.head) dz[tid] = from_float<T>(constant ? value : gradient_at(g, to_float<T>(z[tid]), k));
        const int c = r.element(r.n_vec) + tid;
        if (stretch == n_stretches - 1 && tid < r.tail)
            dz[c] = from_float<T>(constant ? value : gradient_at(g, to_float<T>(z[c]), k));
    } else {                                                                        // the two rows are aligned differently
        from = min(n_classes, stretch * kStretch * N);
        to = stretch == n_stretches - 1 ? n_classes : min(n_classes, from + kStretch * N);
        for (int c = from + tid; c < to; c += kRowThreads)
            dz[c] = from_float<T>(constant ? value : gradient_at(g, to_float<T>(z[c]), k));
    }
    if (constant) return;
    __syncthreads();                                                                // the stretch is written before the given classes
    if (tid < 1 + (in.top ? n_top : 0)) given_class<T>(g, in, top_indices, z, dz, row, n_top, tid, from, to, inv_t, k);
}

// ---- host side -------------------------------------------------------------------------------------------------------
int multiprocessors(int* n) {
    int device;
    GMC_CUDA_TRY(cudaGetDevice(&device));
    GMC_CUDA_TRY(cudaDeviceGetAttribute(n, cudaDevAttrMultiProcessorCount, device));
    return GMC_OK;
}

template <typename T>
int forward_typed(const void* logits, const long long* targets, long long n_rows, int n_classes, long long row_stride, float inv_t,
                  long long ignored, int n_top, const Outputs& out, cudaStream_t stream) {
    const T* z = static_cast<const T*>(logits);
    const float k = kLog2e * inv_t;
    if (n_classes <= kSmallClasses) {
        const unsigned grid = unsigned((n_rows + kSmallThreads / 32 - 1) / (kSmallThreads / 32));
#define GMC_SMALL(E)                                                                                                         \
    forward_small_kernel<T, E><<<grid, kSmallThreads, 0, stream>>>(z, targets, n_rows, n_classes, row_stride, inv_t, k, ignored, n_top, out)
        if (n_classes <= 32) GMC_SMALL(1);
        else if (n_classes <= 64) GMC_SMALL(2);
        else if (n_classes <= 128) GMC_SMALL(4);
        else if (n_classes <= 256) GMC_SMALL(8);
        else if (n_classes <= 512) GMC_SMALL(16);
        else GMC_SMALL(32);
#undef GMC_SMALL
        GMC_LAUNCH_CHECK();
        return GMC_OK;
    }
    int n_sm = 0;
    if (int s = multiprocessors(&n_sm)) return s;
    // a row over several CTAs while there are fewer CTAs than the GPU holds and each keeps a full stretch of vectors (1021 rows
    // of 100003 in fp32: 112 us with one CTA per row, 136 with four, whose alternatives take longer than their columns)
    int n_ranks = 1;
    while (n_ranks < 8 && n_rows * n_ranks < 4LL * n_sm && n_classes / (2 * n_ranks) >= kRowThreads * Vec<T>::N) n_ranks *= 2;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(unsigned(n_rows * n_ranks));
    config.blockDim = dim3(kRowThreads);
    config.stream = stream;
    cudaLaunchAttribute attribute;
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = unsigned(n_ranks);
    attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    if (n_top > 0)
        GMC_CUDA_TRY(cudaLaunchKernelEx(&config, forward_row_kernel<T, true>, z, targets, n_classes, row_stride, n_ranks, inv_t, k, ignored, n_top, out));
    else
        GMC_CUDA_TRY(cudaLaunchKernelEx(&config, forward_row_kernel<T, false>, z, targets, n_classes, row_stride, n_ranks, inv_t, k, ignored, n_top, out));
    return GMC_OK;
}

template <typename T>
int backward_typed(const void* logits, const long long* targets, const long long* top_indices, const float* stats, const float* entropy,
                   const Incoming& in, void* grad, long long n_rows, int n_classes, long long row_stride, float inv_t, long long ignored,
                   int n_top, cudaStream_t stream) {
    const T* z = static_cast<const T*>(logits);
    T* dz = static_cast<T*>(grad);
    const float k = kLog2e * inv_t;
    if (n_classes <= kSmallClasses) {
        const unsigned grid = unsigned((n_rows + kSmallThreads / 32 - 1) / (kSmallThreads / 32));
#define GMC_SMALL(E)                                                                                                              \
    backward_small_kernel<T, E><<<grid, kSmallThreads, 0, stream>>>(z, targets, top_indices, stats, entropy, in, dz, n_rows,      \
                                                                    n_classes, row_stride, inv_t, k, ignored, n_top)
        if (n_classes <= 32) GMC_SMALL(1);
        else if (n_classes <= 64) GMC_SMALL(2);
        else if (n_classes <= 128) GMC_SMALL(4);
        else if (n_classes <= 256) GMC_SMALL(8);
        else if (n_classes <= 512) GMC_SMALL(16);
        else GMC_SMALL(32);
#undef GMC_SMALL
    } else {
        const int n_stretches = (n_classes + kStretch * Vec<T>::N - 1) / (kStretch * Vec<T>::N);
        if (n_rows * n_stretches > 0x7fffffffLL) return GMC_ERR_BAD_DIMS;
        backward_row_kernel<T><<<unsigned(n_rows * n_stretches), kRowThreads, 0, stream>>>(z, targets, top_indices, stats, entropy, in, dz, n_stretches,
                                                                                           n_classes, row_stride, inv_t, k, ignored, n_top);
    }
    GMC_LAUNCH_CHECK();
    return GMC_OK;
}

int check_sizes(int dtype, long long n_rows, long long n_classes, long long row_stride, float temperature, int n_top) {
    if (n_rows < 0 || n_classes < 1 || n_classes > (1LL << 30) || row_stride < 0) return GMC_ERR_BAD_DIMS;
    if (n_rows > (1LL << 27)) return GMC_ERR_BAD_DIMS;                              // grid of short rows and of clusters of eight
    if (dtype < GMC_FLOAT32 || dtype > GMC_FLOAT16) return GMC_ERR_UNSUPPORTED;
    if (!(temperature >= kMinTemperature && temperature <= kMaxTemperature)) return GMC_ERR_UNSUPPORTED;
    if (n_top < 0 || n_top > kMaxTop || n_top > n_classes) return GMC_ERR_UNSUPPORTED;
    return GMC_OK;
}

}  // namespace
}  // namespace gmc

GMC_DEFINE_TU_CHECK_WORD(log_probabilities)

extern "C" int gmc_log_probabilities_forward(const void* logits, int dtype, const long long* targets, long long n_rows,
                                             long long n_classes, long long row_stride, float temperature, long long ignore_index,
                                             int n_top, float* target, float* entropy, float* stats, float* top,
                                             long long* top_indices, void* stream) {
    using namespace gmc;
    if (int s = check_sizes(dtype, n_rows, n_classes, row_stride, temperature, n_top)) return s;
    if (n_rows == 0) return GMC_OK;
    if (!logits || !entropy || (targets == nullptr) != (target == nullptr)) return GMC_ERR_NULL_POINTER;
    if (n_top > 0 && (!top || !top_indices)) return GMC_ERR_NULL_POINTER;
    const Outputs out = {target, entropy, stats, top, top_indices};
    const int c = int(n_classes);
    const float inv_t = 1.f / temperature;
    cudaStream_t s = as_stream(stream);
    if (dtype == GMC_FLOAT32) return forward_typed<float>(logits, targets, n_rows, c, row_stride, inv_t, ignore_index, n_top, out, s);
    if (dtype == GMC_BFLOAT16) return forward_typed<__nv_bfloat16>(logits, targets, n_rows, c, row_stride, inv_t, ignore_index, n_top, out, s);
    return forward_typed<__half>(logits, targets, n_rows, c, row_stride, inv_t, ignore_index, n_top, out, s);
}

extern "C" int gmc_log_probabilities_backward(const void* logits, int dtype, const long long* targets, const long long* top_indices,
                                              const float* stats, const float* entropy, const float* grad_target,
                                              const float* grad_entropy, const float* grad_top, void* grad_logits, long long n_rows,
                                              long long n_classes, long long row_stride, float temperature, long long ignore_index,
                                              int n_top, void* stream) {
    using namespace gmc;
    if (int s = check_sizes(dtype, n_rows, n_classes, row_stride, temperature, n_top)) return s;
    if (n_rows == 0) return GMC_OK;
    if (!logits || !stats || !entropy || !grad_logits || (grad_target && !targets)) return GMC_ERR_NULL_POINTER;
    if (grad_top && (n_top == 0 || !top_indices)) return GMC_ERR_NULL_POINTER;
    const Incoming in = {grad_target, grad_entropy, grad_top};
    const int c = int(n_classes);
    const float inv_t = 1.f / temperature;
    cudaStream_t s = as_stream(stream);
    if (dtype == GMC_FLOAT32)
        return backward_typed<float>(logits, targets, top_indices, stats, entropy, in, grad_logits, n_rows, c, row_stride, inv_t, ignore_index, n_top, s);
    if (dtype == GMC_BFLOAT16)
        return backward_typed<__nv_bfloat16>(logits, targets, top_indices, stats, entropy, in, grad_logits, n_rows, c, row_stride, inv_t, ignore_index, n_top, s);
    return backward_typed<__half>(logits, targets, top_indices, stats, entropy, in, grad_logits, n_rows, c, row_stride, inv_t, ignore_index, n_top, s);
}
