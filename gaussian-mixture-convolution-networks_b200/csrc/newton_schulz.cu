// Orthogonalisation of updates by Newton-Schulz products, and the Muon update around it.
//
//   X = U / (|U| + eps) (transposed if it is taller than wide);  steps times: A = X X^T, B = b A + c A A, X <- a X + B X
//
// Precision. The polynomial multiplies what is small by up to a^steps (485 for the usual coefficients), and rounding errors
// with it, so operands of 11 or 8 bits would leave errors of 1e-1 where U is close to rank one. Every operand is therefore
// held as two fp16 planes, value = hi + lo (22 bits; scaled by a power of two, which the bound of the polynomial on
// [0, 1] keeps below the largest fp16 number), and a product takes three tensor-core products, hi hi + hi lo + lo hi, into
// one fp32 accumulator; the left-out lo lo is 2^-22 of it. The cost is three times the operations of one product.
//
// Layout. Both planes lie in global memory as blocks of 128 rows x 64 columns in the exact byte order the tensor core reads
// from shared memory (128-byte swizzle, eight rows of hi and of lo in turn), padded with zeros: loading an operand tile is
// one or two contiguous bulk copies, whatever the matrix's shape (a copy costs its issuing thread 130 cycles or more, whatever
// its size), and X serves both as rows (X X^T, K = columns) and across (P X, K = rows) without a transposed copy.
// A and A A are symmetric: only tiles on and below the diagonal are computed and stored, what lies above is read across.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "tcgen05.cuh"

namespace gmc {
namespace {

namespace cg = cooperative_groups;

constexpr int kPairs = 74;                       // CTA pairs of the GPU: 148 multiprocessors
constexpr int kMaxMatrices = 48;                 // descriptors of one launch (kernel parameter)
constexpr int kBlockBytes = 2 * 128 * 64 * 2;    // one block, both planes
constexpr int kHalfBlock = kBlockBytes / 2;      // 64 rows of it
constexpr int kStageBytes = 2 * kBlockBytes;     // both operands, 64 wide in K
constexpr int kStages = 3;
constexpr int kWarpRows = kBlockBytes / 4;       // a writing warp's 32 rows of a block
constexpr int kChainSmem = kStages * kStageBytes + 1024;
constexpr int kWholeAxis = 1 << 20;              // Matrix::chunk: one accumulation, whatever the axis
constexpr int kWholeStages = 32, kLongChunk = 16;    // 16-bit results: the longest such axis, and the chunk beyond it
constexpr float kScaleX = 32768.f;               // |X| stays below 1.8, the largest fp16 number is 65504
constexpr int kNormElements = 4096;              // elements of a matrix per CTA of the norm

// The matrices of a launch. Wide form: m <= n after the transposition.
struct Matrix {
    const void* update;         // [rows, cols], unit column stride
    float* momentum;            // [rows, cols] contiguous, or null
    void* out;                  // [rows, cols], unit column stride: the orthogonalised update, or the parameters
    long long update_stride, out_stride;
    int rows, cols;
    int row_tiles, col_blocks;  // of the wide form: 128 rows, 64 columns (even number)
    float rate;                 // factor of the orthogonalised update that is subtracted from the parameters
    int norm_first, block_first;                       // first CTA of the matrix in the launches before and after the chain
    int pair_first, pairs;                             // CTA pairs of the matrix in the chain
    int gram_wide, poly_wide, step_wide, splits;       // tiles 256 instead of 128 columns wide; shares of the columns in X X^T
    int chunk;                                         // stages, 64 wide in K each, that are added up in the tensor core
    long long x_block, gram_block, partial_first;      // first block, first partial sum in the workspace's arrays
};
struct Batch {
    Matrix m[kMaxMatrices];
    int n;
    __half *x[2], *gram, *poly;
    double* squares;            // one per CTA of the norm
    float* partial;             // tiles of X X^T over shares of the columns
    unsigned* arrived;          // one counter per matrix, then the failure flag
    int norm_ctas, pairs, blocks;
    bool whole;                 // every matrix has chunk = kWholeAxis
    int lost_wait;              // writing warp of the launch whose first wait counts as run out (a test's), or -1
};
struct Momentum {
    float beta, one_minus_beta;
    int nesterov;
    float decay;                // factor of the parameters
};

template <int Matrix::*FIRST>
__device__ __forceinline__ int find_matrix(const Batch& b, int cta) {
    int i = 0;
    while (i + 1 < b.n && cta >= b.m[i + 1].*FIRST) ++i;
    return i;
}

// Eight neighbouring elements, with vector accesses where `aligned` says that their address allows them.
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool aligned, float (&v)[8]) {
    if (aligned) {
        constexpr int N = 16 / int(sizeof(T));
        union { uint4 raw[8 / N]; T e[8]; } u;
#pragma unroll
        for (int i = 0; i < 8 / N; ++i) u.raw[i] = reinterpret_cast<const uint4*>(p)[i];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = float(u.e[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = float(p[e]);
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, bool aligned, const float (&v)[8]) {
    if (aligned) {
        constexpr int N = 16 / int(sizeof(T));
        union { uint4 raw[8 / N]; T e[8]; } u;
#pragma unroll
        for (int e = 0; e < 8; ++e) u.e[e] = T(v[e]);
#pragma unroll
        for (int i = 0; i < 8 / N; ++i) reinterpret_cast<uint4*>(p)[i] = u.raw[i];
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = T(v[e]);
    }
}
__device__ __forceinline__ bool rows_aligned(const void* p, long long stride, int size) {
    return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t(stride) * size)) & 15u) == 0;
}

// Sum of squares of kNormElements elements per CTA, in fp64 (the squares of small updates leave the fp32 range); with a
// momentum the running average is updated on the way. 2048 x 2048 in fp32: 9 us, 1.9 TB/s with cold caches, most of it launch
// and latency; 59 MB of updates and momenta: 16 us, 3.7 TB/s read and as much again written.
template <typename T, bool MUON>
__global__ void __launch_bounds__(256) norm_kernel(const __grid_constant__ Batch b, Momentum mo) {
    if (blockIdx.x == 0 && threadIdx.x <= unsigned(b.n)) b.arrived[threadIdx.x] = 0;        // for the chain
    const int which = find_matrix<&Matrix::norm_first>(b, blockIdx.x);
    const Matrix& m = b.m[which];
    const long long total = (long long)m.rows * m.cols;
    const long long first = (long long)(int(blockIdx.x) - m.norm_first) * kNormElements;
    const int count = int(min((long long)kNormElements, total - first));
    double s = 0.;
    // the update's element and the momentum's at the same place
    auto blend = [&](float u, float& old) {
        old = mo.beta * old + mo.one_minus_beta * u;
        return mo.nesterov ? mo.one_minus_beta * u + mo.beta * old : old;
    };
    const T* update = static_cast<const T*>(m.update);
    if (m.update_stride == m.cols && rows_aligned(update, 0, 1) && (!MUON || rows_aligned(m.momentum, 0, 1))) {
        // one row as far as the norm is concerned
#pragma unroll 2
        for (int i = threadIdx.x * 8; i < count; i += 256 * 8) {
            float u[8], old[8];
            if (i + 8 <= count) {
                load8(update + first + i, true, u);
                if constexpr (MUON) {
                    load8(m.momentum + first + i, true, old);
#pragma unroll
                    for (int e = 0; e < 8; ++e) u[e] = blend(u[e], old[e]);
                    store8(m.momentum + first + i, true, old);
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) s += double(u[e]) * double(u[e]);
            } else {
                for (int e = i; e < count; ++e) {
                    float v = float(update[first + e]);
                    if constexpr (MUON) v = blend(v, m.momentum[first + e]);
                    s += double(v) * double(v);
                }
            }
        }
    } else {
        const int row0 = int(first / m.cols), col0 = int(first - (long long)row0 * m.cols);
        const unsigned cols = unsigned(m.cols);
#pragma unroll 4
        for (int i = threadIdx.x; i < count; i += 256) {
            const unsigned at = unsigned(col0 + i), r = at / cols;
            float u = float(update[(row0 + (long long)r) * m.update_stride + (at - r * cols)]);
            if constexpr (MUON) u = blend(u, m.momentum[first + i]);
            s += double(u) * double(u);
        }
    }
    __shared__ double warp_sum[8];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0) warp_sum[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; ++w) s += warp_sum[w];
        b.squares[blockIdx.x] = s;
    }
}

union Chunk {
    uint4 raw;
    __half h[8];
};

// Eight columns: v c1, plus c0 (in_hi + in_lo), as planes.
template <bool ADD>
__device__ __forceinline__ void split8(const float* v, float c1, float c0, const uint4& in_hi, const uint4& in_lo, uint4& hi, uint4& lo) {
    const __half2* ih = reinterpret_cast<const __half2*>(&in_hi);
    const __half2* il = reinterpret_cast<const __half2*>(&in_lo);
    __half2* oh = reinterpret_cast<__half2*>(&hi);
    __half2* ol = reinterpret_cast<__half2*>(&lo);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float x = v[2 * e] * c1, y = v[2 * e + 1] * c1;
        if (ADD) {
            const float2 h = __half22float2(ih[e]), l = __half22float2(il[e]);
            x += c0 * (h.x + l.x);
            y += c0 * (h.y + l.y);
        }
        oh[e] = __floats2half2_rn(x, y);
        const float2 back = __half22float2(oh[e]);
        ol[e] = __floats2half2_rn(x - back.x, y - back.y);
    }
}

// X = U / (|U| + eps) as planes: one 128 x 64 block per CTA, padding included: 2048 x 2048 in fp32
// 11 us (cold caches; 2.9 TB/s of 17 MB in and 17 MB out), 4095 x 6001 in bf16, where rows start anywhere, 42 us. Bound by the
// latency of one block per CTA: update -> shared memory -> copy.
template <typename T, bool MUON>
__global__ void __launch_bounds__(256) split_kernel(const __grid_constant__ Batch b, Momentum mo, float epsilon) {
    const int which = find_matrix<&Matrix::block_first>(b, blockIdx.x);
    const Matrix& m = b.m[which];
    const int block = int(blockIdx.x) - m.block_first;
    const int norm_end = which + 1 < b.n ? b.m[which + 1].norm_first : b.norm_ctas;
    __shared__ double warp_sum[8];
    double s = 0.;
    for (int i = m.norm_first + threadIdx.x; i < norm_end; i += 256) s += b.squares[i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0) warp_sum[threadIdx.x >> 5] = s;
    __syncthreads();
    s = 0.;
    for (int w = 0; w < 8; ++w) s += warp_sum[w];
    const float factor = float(double(kScaleX) / (sqrt(s) + double(epsilon)));        // the norm itself may leave the fp32 range
    const bool tall = m.rows > m.cols;
    const int wide_rows = tall ? m.cols : m.rows, wide_cols = tall ? m.rows : m.cols;
    const int row_tile = block / m.col_blocks, col_block = block - row_tile * m.col_blocks;
    // The block is laid out in shared memory, where its bytes' order costs nothing, and leaves as one bulk copy.
    __shared__ __align__(128) uint8_t image[kBlockBytes];
    const T* update = static_cast<const T*>(m.update);
    const bool vectors = rows_aligned(update, m.update_stride, sizeof(T)), momentum_vectors = rows_aligned(m.momentum, m.cols, 4);
    const uint4 none = {};
#pragma unroll 2
    for (int i = threadIdx.x; i < 128 * 8; i += 256) {
        const int row = tall ? i & 127 : i >> 3, chunk = tall ? i >> 7 : i & 7;      // neighbouring threads read along a row
        const int r = row_tile * 128 + row, c = col_block * 64 + chunk * 8;
        float u[8], old[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = old[e] = 0.f;
        if (!tall && r < wide_rows && c + 8 <= wide_cols) {
            load8(update + r * m.update_stride + c, vectors, u);
            if constexpr (MUON) load8(m.momentum + (long long)r * m.cols + c, momentum_vectors, old);
        } else if (r < wide_rows) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (c + e < wide_cols) {
                    const long long rr = tall ? c + e : r, cc = tall ? r : c + e;
                    u[e] = float(update[rr * m.update_stride + cc]);
                    if constexpr (MUON) old[e] = m.momentum[rr * m.cols + cc];
                }
            }
        }
        if constexpr (MUON) {
#pragma unroll
            for (int e = 0; e < 8; ++e) u[e] = mo.nesterov ? mo.one_minus_beta * u[e] + mo.beta * old[e] : old[e];
        }
        uint4 hi, lo;
        split8<false>(u, factor, 0.f, none, none, hi, lo);
        uint8_t* at = image + swizzled_offset(row, chunk);
        *reinterpret_cast<uint4*>(at) = hi;
        *reinterpret_cast<uint4*>(at + kPlaneOffset) = lo;
    }
    fence_proxy_async();
    __syncthreads();
    if (threadIdx.x == 0) {
        uint8_t* to = reinterpret_cast<uint8_t*>(b.x[0]) + (m.x_block + block) * kBlockBytes;
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(to), "r"(smem_u32(image)), "n"(kBlockBytes) : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
}

// The last X as the output's type, or subtracted from the parameters. 2048 x 2048 in fp32: 11 us, 3 TB/s read and written
// together; bound, as split_kernel, by the latency of one block per CTA.
template <typename T, bool MUON>
__global__ void __launch_bounds__(256) finish_kernel(const __grid_constant__ Batch b, Momentum mo, int which_x) {
    const int which = find_matrix<&Matrix::block_first>(b, blockIdx.x);
    const Matrix& m = b.m[which];
    const int block = int(blockIdx.x) - m.block_first;
    const bool tall = m.rows > m.cols;
    const int wide_rows = tall ? m.cols : m.rows, wide_cols = tall ? m.rows : m.cols;
    const int row_tile = block / m.col_blocks, col_block = block - row_tile * m.col_blocks;
    __shared__ __align__(128) uint8_t image[kBlockBytes];
    __shared__ uint64_t arrived;
    if (threadIdx.x == 0) {
        mbar_init(&arrived, 1);
        fence_mbar_init();
        mbar_arrive_expect_tx(&arrived, kBlockBytes);
        bulk_copy_g2s(image, reinterpret_cast<const uint8_t*>(b.x[which_x]) + (m.x_block + block) * kBlockBytes, kBlockBytes, &arrived);
    }
    T* out = static_cast<T*>(m.out);
    const bool vectors = rows_aligned(out, m.out_stride, sizeof(T));
    __syncthreads();
    const bool ok = mbar_wait_bounded(&arrived, 0) && b.arrived[b.n] == 0;
    if (!tall && !vectors) {
        // rows that start anywhere: single elements, neighbouring threads along a row (4095 x 6001 in bf16: 40 us, and 87 with
        // eight elements per thread; reading in that way gained nothing in split_kernel, 52 us and 42)
#pragma unroll 8
        for (int i = threadIdx.x; i < 128 * 64; i += 256) {
            const int row = i >> 6, col = i & 63, r = row_tile * 128 + row, c = col_block * 64 + col;
            if (r >= wide_rows || c >= wide_cols) continue;
            const uint8_t* at = image + swizzled_offset(row, col >> 3) + (col & 7) * 2;
            float v = (__half2float(*reinterpret_cast<const __half*>(at)) + __half2float(*reinterpret_cast<const __half*>(at + kPlaneOffset))) *
                      (1.f / kScaleX);
            if (!ok) v = __int_as_float(0x7fffffff);
            T* to = out + r * m.out_stride + c;
            *to = T(MUON ? float(*to) * mo.decay - m.rate * v : v);
        }
        return;
    }
#pragma unroll 2
    for (int i = threadIdx.x; i < 128 * 8; i += 256) {
        const int row = tall ? i & 127 : i >> 3, chunk = tall ? i >> 7 : i & 7;
        const int r = row_tile * 128 + row, c = col_block * 64 + chunk * 8;
        if (r >= wide_rows || c >= wide_cols) continue;
        const uint8_t* at = image + swizzled_offset(row, chunk);
        Chunk hi, lo;
        hi.raw = *reinterpret_cast<const uint4*>(at);
        lo.raw = *reinterpret_cast<const uint4*>(at + kPlaneOffset);
        float v[8], old[8];
        const bool whole = !tall && c + 8 <= wide_cols;
        if (MUON && whole) load8(out + r * m.out_stride + c, true, old);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[e] = (__half2float(hi.h[e]) + __half2float(lo.h[e])) * (1.f / kScaleX);
            if (!ok) v[e] = __int_as_float(0x7fffffff);
            if (MUON && whole) v[e] = old[e] * mo.decay - m.rate * v[e];
        }
        if (whole) {
            store8(out + r * m.out_stride + c, true, v);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (c + e < wide_cols) {
                    T* to = out + (tall ? (c + e) * m.out_stride + r : r * m.out_stride + c + e);
                    *to = T(MUON ? float(*to) * mo.decay - m.rate * v[e] : v[e]);
                }
            }
        }
    }
}

// All products of a call in one persistent launch. A matrix has some pairs of CTAs; a pair computes tiles of 256 rows (128
// per CTA) by 256 or 128 columns with two-CTA MMAs, which read half the operand bytes per CTA that one CTA alone would (with
// one CTA and 128 x 128 tiles the shared memory's 128 bytes per cycle, filled and read at once, held the tensor core at 40 %).
// Between the products of a step the matrix's CTAs wait for one another at a counter in global memory; the launch is
// cooperative, so all of them are resident.
//
// Roles: warps 0-7 write tiles (warp w: rows 32 (w % 4) .. + 31 of the CTA's 128, half w / 4 of the columns), warps 8 and 9
// load one operand each (bulk copies into a ring of stages), warps 10 and 11 of the pair's first CTA issue the MMAs of the
// mixed products and of hi hi (issuing one takes its thread 80 cycles, so that one thread would not keep up), warp 10 of
// the second CTA passes on that its operands have arrived. Behind the stages of a tile the ring carries one or two more,
// with what the epilogue adds (A for B, X for the next X): the writers put the result in their place, from where it leaves
// as contiguous bulk copies.
//
// The tensor core adds into its fp32 accumulator without rounding to nearest: the sums fall short by about n 2^-24 of
// themselves after n additions. For fp32 results hi hi is therefore accumulated over two to eight stages (128 to 512 in K,
// 8 to 32 additions, by the matrix's size) only and then added to registers, while other MMAs run, with the mean of the loss
// made good; hi lo and lo hi, 2^-11 as large, have an accumulator of their own. Where results are rounded to 16 bits and no
// sum is longer than 2048, one accumulation takes the whole axis, and both sums are ready and read at the same time.
//
// Measured (fp32, five steps, the launches around the chain included): 4095 x 6001 in bf16 5.46 ms, 339 TFLOP/s of the
// polynomial's and 1018 of the tensor core's products, 0.72 of a large library product under the same power limit; bound by
// the MMAs (a stage takes 1516 cycles, its MMAs 1536 at the nominal rate), by the sums' way out every 16 stages (1400) and by the
// last tiles of a product, for which the other pairs wait. 2048 x 2048: 678 us, 253 TFLOP/s; fp32 sums leave the tensor core
// every 512 in K, and 256 bytes a thread of the chunked form's registers spill (none of the whole form's). Below about 1000 rows
// the latencies of a product (barrier, first loads, one tile's way out: 11 to 13 us) count for more than its MMAs.
enum Product { GRAM, POLY, STEP };
constexpr int kWriters = 256;
constexpr int kChainThreads = kWriters + 128;
constexpr int kMixedColumns = 256;                // TMEM columns: 256 for hi hi, 256 for the mixed products

// A matrix in the workspace: blocks of 128 x 64, both planes.
struct Planes {
    uint8_t* base;
    int row_blocks, col_blocks;
    __device__ __forceinline__ uint8_t* block(int r, int c) const { return base + ((long long)r * col_blocks + c) * kBlockBytes; }
};

// One operand of a stage: `groups` x 64 rows from row group `row` on, 64 wide in K at `kb`. Along K the rows are those of the
// matrix; across K they are its columns (K = its rows).
__device__ __forceinline__ void load_operand(uint8_t* to, const Planes& p, int row, int groups, int kb, bool across, uint64_t* bar) {
    if (!across) {
        const int r = min(row >> 1, p.row_blocks - 1);                                  // rows behind the last tile are not stored
        bulk_copy_g2s(to, p.block(r, kb) + (groups == 1 ? (row & 1) * kHalfBlock : 0), groups * kHalfBlock, bar);
    } else {
        for (int g = 0; g < groups; ++g)
            bulk_copy_g2s(to + g * kHalfBlock, p.block(kb >> 1, min(row + g, p.col_blocks - 1)) + (kb & 1) * kHalfBlock, kHalfBlock, bar);
    }
}

// Tiles of a symmetric product: rows of 256, columns of 256 or 128, the column's 256 not above the row's.
__host__ __device__ __forceinline__ int symmetric_tiles(int row_tiles, int wide) {
    const int rows = (row_tiles + 1) / 2;
    return wide ? rows * (rows + 1) / 2 : rows * (rows + 1) - (row_tiles & 1);
}
__device__ __forceinline__ void symmetric_tile(int tile, int wide, int& ti, int& tj) {
    ti = 0;
    if (wide) {
        ti = int((sqrtf(8.f * float(tile) + 1.f) - 1.f) * 0.5f);
        while (ti * (ti + 1) / 2 > tile) --ti;
        while ((ti + 1) * (ti + 2) / 2 <= tile) ++ti;
        tj = tile - ti * (ti + 1) / 2;
    } else {
        ti = int((sqrtf(4.f * float(tile) + 1.f) - 1.f) * 0.5f);
        while (ti * (ti + 1) > tile) --ti;
        while ((ti + 1) * (ti + 2) <= tile) ++ti;
        tj = tile - ti * (ti + 1);
    }
}

// What a CTA needs to walk through the products of its matrix; the same in every role.
struct Walk {
    Planes x0, x1, gram, poly;
    int pair, pairs, splits;
    int gram_wide, poly_wide, step_wide;
    __device__ __forceinline__ const Planes& x(int i) const { return i ? x1 : x0; }
    __device__ __forceinline__ int wide(Product p) const { return p == GRAM ? gram_wide : p == POLY ? poly_wide : step_wide; }
    __device__ __forceinline__ int tiles(Product p) const {
        return p == STEP ? ((gram.row_blocks + 1) / 2) * ((x0.col_blocks + (step_wide ? 3 : 1)) / (step_wide ? 4 : 2))
                         : symmetric_tiles(gram.row_blocks, wide(p));
    }
    // unit -> tile row (256), tile column (256 or 128), first and last 64 in K
    __device__ __forceinline__ void unit(Product p, int u, int& ti, int& tj, int& k0, int& k1) const {
        const int n = tiles(p), share = u / n, tile = u - share * n, all = p == GRAM ? x0.col_blocks : gram.col_blocks;
        if (p == STEP) {
            const int columns = (x0.col_blocks + (step_wide ? 3 : 1)) / (step_wide ? 4 : 2);
            ti = tile / columns;
            tj = tile - ti * columns;
        } else {
            symmetric_tile(tile, wide(p), ti, tj);
        }
        const int parts = p == GRAM ? splits : 1;
        k0 = int((long long)all * share / parts);
        k1 = int((long long)all * (share + 1) / parts);
    }
    // stages behind a tile's own: what is added to its sums, and the place where the result is laid out
    __device__ __forceinline__ int extra(Product p) const { return p == GRAM && splits > 1 ? 0 : wide(p) ? 2 : 1; }
    __device__ __forceinline__ int units(Product p) const { return tiles(p) * (p == GRAM ? splits : 1); }
};

__device__ __forceinline__ bool wait_counter(const unsigned* counter, unsigned value) {
    for (int i = 0; i < (1 << 22); ++i) {
        unsigned now;
        asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(now) : "l"(counter) : "memory");
        if (now >= value) return true;
    }
    report_check(CHECK_MBARRIER_TIMEOUT);
    return false;
}
__device__ __forceinline__ void fence_proxy_async_all() { asm volatile("fence.proxy.async;" ::: "memory"); }
__device__ __forceinline__ void writers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kWriters) : "memory"); }

struct ChainBarriers {
    uint64_t full[kStages], peer_full[kStages], empty[kStages], ready[2], drained[2], mixed_ready, mixed_drained, done;
};

// One lane polls for its warp. What it has acquired holds for the other lanes from the barrier on; a shuffle alone orders no
// memory, and they go on to read what other threads, or copies, have written.
__device__ __forceinline__ bool to_warp(bool ok) {
    const int all = __shfl_sync(0xffffffffu, int(ok), 0);
    __syncwarp();
    return all != 0;
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, unsigned parity) {
    bool ok = true;
    if ((threadIdx.x & 31) == 0) ok = mbar_wait_bounded(bar, parity);
    return to_warp(ok);
}

// Writers: the tiles of one product. `tile`, `k` count the tiles and stages since the launch, `phase` has a bit per place of a
// chunk's sums. Narrow tiles leave 128 columns of tensor memory for a second place, taken by every other chunk of a tile, which
// is summed up while the next one is multiplied; in a wide tile the MMAs wait for it (1400 cycles a chunk).
struct WriterCounts {
    unsigned phase, tile, k;
};
// 64 columns of a row in their place: v c1, plus c0 times what is there. The next chunk is read before this one is written,
// which the compiler could not know to be safe.
__device__ __forceinline__ void place_block(const float* v, uint8_t* rows, bool add, float c0, float c1, int lane) {
    uint4 next_hi = {}, next_lo = {};
    if (add) {
        next_hi = *reinterpret_cast<const uint4*>(rows + swizzled_offset(lane, 0));
        next_lo = *reinterpret_cast<const uint4*>(rows + swizzled_offset(lane, 0) + kPlaneOffset);
    }
#pragma unroll
    for (int g = 0; g < 8; ++g) {
        uint8_t* at = rows + swizzled_offset(lane, g);
        const uint4 in_hi = next_hi, in_lo = next_lo;
        if (g < 7 && add) {
            next_hi = *reinterpret_cast<const uint4*>(rows + swizzled_offset(lane, g + 1));
            next_lo = *reinterpret_cast<const uint4*>(rows + swizzled_offset(lane, g + 1) + kPlaneOffset);
        }
        uint4 hi, lo;
        split8<true>(v + g * 8, c1, c0, in_hi, in_lo, hi, lo);
        *reinterpret_cast<uint4*>(at) = hi;
        *reinterpret_cast<uint4*>(at + kPlaneOffset) = lo;
    }
}
// The stage behind a tile holds two neighbouring blocks of the result, complete once its warps (all, or the four of its half)
// have come here: one copy takes them out. Then the stage is free: its barrier expects the two arrivals that the MMA threads'
// commits make for the others.
__device__ __forceinline__ void send_stage(const Planes& to, int row_block, int col_block, const uint8_t* stage, uint64_t* empty, int wide, int warp,
                                           int lane) {
    fence_proxy_async();
    if (wide) asm volatile("bar.sync %0, 128;" ::"r"(2 + (warp >> 2)) : "memory");
    else writers_sync();
    if (lane == 0 && (warp == 0 || (wide && warp == 4))) {
        const int blocks = row_block < to.row_blocks ? min(2, to.col_blocks - col_block) : 0;
        if (blocks > 0)
            asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(to.block(row_block, col_block)), "r"(smem_u32(stage)),
                         "r"(blocks * kBlockBytes)
                         : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        mbar_arrive(empty);
        mbar_arrive(empty);
    }
    __syncwarp();
}

// WHOLE: one accumulation takes the whole axis. `ok` becomes false when a wait runs out. The warp then goes on without
// waiting: the others meet it at barriers that know no limit, and every access stays where it belongs. The result is
// given up for NaN at the end.
template <bool WHOLE>
__device__ __forceinline__ void write_product(Product p, const Walk& w, ChainBarriers& bar, uint8_t* stages, uint32_t tmem, int cta,
                                              WriterCounts& n, const Planes& to, float c0, float c1, int stages_per_chunk, float* partial,
                                              bool& ok) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
    const int wide = w.wide(p), half = wide ? 128 : 64, col0 = (warp >> 2) * half;
    const int units = w.units(p);
    for (int u = w.pair; u < units; u += w.pairs, ++n.tile) {
        int ti, tj, k0, k1;
        w.unit(p, u, ti, tj, k0, k1);
        const int diagonal = (2 * ti + cta) * 128 + (warp & 3) * 32 + lane - tj * 2 * half - col0;       // this row's
        if constexpr (WHOLE) {
            // 32 columns at a time from tensor memory to their place, nothing kept in registers (with the sums of
            // 128 columns in them the code is four times as long, and the time of a tile with it).
            n.k += k1 - k0;
            const bool shared_out = p == GRAM && w.splits > 1;
            const unsigned k = n.k + (wide ? warp >> 2 : 0), s = k % kStages;
            n.k += w.extra(p);
            ok = ok && warp_wait(&bar.ready[0], n.tile & 1);
            if (!shared_out) ok = ok && warp_wait(&bar.full[s], (k / kStages) & 1);
            tmem_fence_after();
            const float loss = 0x1p-25f * 4.f * float(k1 - k0), made_good = 1.f + 0.7f * loss;
            const float diagonal_good = 1.f + (p == GRAM ? 2.f : p == POLY ? 2.4f : 0.7f) * loss;
#pragma unroll 1
            for (int q = 0; q < half; q += 32) {
                float v[32], mixed[32];
                tmem_load32(tmem + lanes + col0 + q, v, tmem + kMixedColumns + lanes + col0 + q, mixed);
#pragma unroll
                for (int e = 0; e < 32; ++e) v[e] = v[e] * (q + e == diagonal ? diagonal_good : made_good) + mixed[e];
                if (shared_out) {
                    // [unit][CTA][column][row]
                    float* out = partial + (((long long)u * 2 + cta) * (2 * half) + col0 + q) * 128 + (warp & 3) * 32 + lane;
#pragma unroll
                    for (int e = 0; e < 32; ++e) out[e * 128] = v[e];
                    continue;
                }
                uint8_t* rows = stages + s * kStageBytes + (wide ? q >> 6 : warp >> 2) * kBlockBytes + (warp & 3) * kWarpRows;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    uint8_t* at = rows + swizzled_offset(lane, ((q & 63) >> 3) + g);
                    uint4 in_hi = {}, in_lo = {}, hi, lo;
                    if (p != GRAM) {
                        in_hi = *reinterpret_cast<const uint4*>(at);
                        in_lo = *reinterpret_cast<const uint4*>(at + kPlaneOffset);
                    }
                    split8<true>(v + g * 8, c1, c0, in_hi, in_lo, hi, lo);
                    *reinterpret_cast<uint4*>(at) = hi;
                    *reinterpret_cast<uint4*>(at + kPlaneOffset) = lo;
                }
            }
            tmem_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_at(&bar.drained[0], 0);
            if (!shared_out)
                send_stage(to, 2 * ti + cta, (tj * 2 * half + (wide ? col0 : 0)) >> 6, stages + s * kStageBytes, &bar.empty[s], wide, warp, lane);
        } else {
            float sum[128];
#pragma unroll
            for (int i = 0; i < 128; ++i) sum[i] = 0.f;
            unsigned place = 0;
            for (int kb = k0; kb < k1; kb += stages_per_chunk, place ^= wide ? 0 : 1) {
                ok = ok && warp_wait(&bar.ready[place], (n.phase >> place) & 1);
                n.phase ^= 1u << place;
                tmem_fence_after();
                // The mean of what the chunk's n = 4 additions per stage have lost, as measured against 64-bit sums: 2.0 n 2^-25 on the
                // diagonal of X X^T, where all terms have one sign; 2.4 n 2^-25 on A A's, where most of a sum comes with one term;
                // 0.7 n 2^-25 where signs are random (off the diagonals) or one term of B X, the diagonal's, outweighs the others
                // (the half of the additions that follow it lose half a step each).
                const float loss = 0x1p-25f * 4.f * float(min(stages_per_chunk, k1 - kb));
                const float made_good = 1.f + 0.7f * loss, diagonal_good = 1.f + (p == GRAM ? 2.f : p == POLY ? 2.4f : 0.7f) * loss;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    if (q < 2 || wide) {
                        float v[32];
                        tmem_load32(tmem + place * 128 + lanes + col0 + q * 32, v);
#pragma unroll
                        for (int i = 0; i < 32; ++i) sum[q * 32 + i] += v[i] * (q * 32 + i == diagonal ? diagonal_good : made_good);
                    }
                }
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_at(&bar.drained[place], 0);
            }
            ok = ok && warp_wait(&bar.mixed_ready, n.tile & 1);
            tmem_fence_after();
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (q < 2 || wide) {
                    float v[32];
                    tmem_load32(tmem + kMixedColumns + lanes + col0 + q * 32, v);
#pragma unroll
                    for (int i = 0; i < 32; ++i) sum[q * 32 + i] += v[i];
                }
            }
            tmem_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_at(&bar.mixed_drained, 0);
            n.k += k1 - k0;
            if (p == GRAM && w.splits > 1) {
                // [unit][CTA][column][row]
                float* out = partial + (((long long)u * 2 + cta) * (2 * half) + col0) * 128 + (warp & 3) * 32 + lane;
#pragma unroll
                for (int i = 0; i < 128; ++i)
                    if (i < 64 || wide) out[i * 128] = sum[i];
                continue;
            }
            // the stages behind the tile's: two blocks each. Wide: warps 0-3 have the first one's, warps 4-7 the second one's.
            const unsigned k = n.k + (wide ? warp >> 2 : 0), s = k % kStages;
            n.k += wide ? 2 : 1;
            ok = ok && warp_wait(&bar.full[s], (k / kStages) & 1);
            place_block(sum, stages + s * kStageBytes + (wide ? 0 : warp >> 2) * kBlockBytes + (warp & 3) * kWarpRows, p != GRAM, c0, c1, lane);
            if (wide) place_block(sum + 64, stages + s * kStageBytes + kBlockBytes + (warp & 3) * kWarpRows, p != GRAM, c0, c1, lane);
            send_stage(to, 2 * ti + cta, (tj * 2 * half + (wide ? col0 : 0)) >> 6, stages + s * kStageBytes, &bar.empty[s], wide, warp, lane);
        }
    }
}

// Writers: adds up the shares of X X^T, 32 rows x 32 columns per warp at a time, in the shares' order.
__device__ __forceinline__ void reduce_gram(const Walk& w, int cta, const float* partial, const Planes& to, float c1) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int columns = w.gram_wide ? 256 : 128, strips = columns / 32, tiles = w.tiles(GRAM);
    for (int i = (w.pair * 2 + cta) * (kWriters / 32) + warp; i < tiles * 2 * strips * 4; i += w.pairs * 2 * (kWriters / 32)) {
        const int quarter = i & 3, strip = (i >> 2) % strips, half = (i >> 2) / strips, of = half & 1, tile = half >> 1;
        int ti, tj;
        symmetric_tile(tile, w.gram_wide, ti, tj);
        const int row_block = 2 * ti + of, col = tj * columns + strip * 32;
        if (row_block >= to.row_blocks || (col >> 6) >= to.col_blocks) continue;
        float v[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) v[c] = 0.f;
        for (int s = 0; s < w.splits; ++s) {
            const float* from = partial + ((((long long)s * tiles + tile) * 2 + of) * columns + strip * 32) * 128 + quarter * 32 + lane;
#pragma unroll
            for (int c = 0; c < 32; ++c) v[c] += from[c * 128];
        }
        uint8_t* out = to.block(row_block, col >> 6) + quarter * kWarpRows;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            uint4 none = {}, hi, lo;
            split8<false>(v + g * 8, c1, 0.f, none, none, hi, lo);
            uint8_t* at = out + swizzled_offset(lane, ((col & 63) >> 3) + g);
            *reinterpret_cast<uint4*>(at) = hi;
            *reinterpret_cast<uint4*>(at + kPlaneOffset) = lo;
        }
    }
}

// The numbers of a step: a product's sums times `factor`, plus `from` times what was there. Without c (two coefficients)
// X X^T gives the polynomial at once and there is no second product.
struct Polynomial {
    float gram_factor, poly_factor, poly_from, step_factor, step_from;
    int linear;
};

template <bool WHOLE>
__global__ void __launch_bounds__(kChainThreads, 1) chain_kernel(const __grid_constant__ Batch b, int steps, Polynomial poly) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ ChainBarriers bar;
    __shared__ uint32_t tmem_address;
    const uint32_t pad = (1024u - (smem_u32(smem_raw) & 1023u)) & 1023u;
    uint8_t* stages = smem_raw + pad;
    const int tid = threadIdx.x, warp = tid >> 5;
    cg::cluster_group cluster = cg::this_cluster();
    const int cta = int(cluster.block_rank()), pair = int(blockIdx.x >> 1);
    const int which = find_matrix<&Matrix::pair_first>(b, pair);
    const Matrix& m = b.m[which];

    __shared__ Walk w;                                                // not in registers: the writers' are full of sums
    if (tid == 0) {
        w.x0 = {reinterpret_cast<uint8_t*>(b.x[0]) + m.x_block * kBlockBytes, m.row_tiles, m.col_blocks};
        w.x1 = {reinterpret_cast<uint8_t*>(b.x[1]) + m.x_block * kBlockBytes, m.row_tiles, m.col_blocks};
        w.gram = {reinterpret_cast<uint8_t*>(b.gram) + m.gram_block * kBlockBytes, m.row_tiles, 2 * m.row_tiles};
        w.poly = {reinterpret_cast<uint8_t*>(b.poly) + m.gram_block * kBlockBytes, m.row_tiles, 2 * m.row_tiles};
        w.pair = pair - m.pair_first;
        w.pairs = m.pairs;
        w.splits = m.splits;
        w.gram_wide = m.gram_wide;
        w.poly_wide = m.poly_wide;
        w.step_wide = m.step_wide;
    }
    unsigned* counter = b.arrived + which;
    unsigned* failed = b.arrived + b.n;
    float* partial = b.partial + m.partial_first;
    const unsigned ctas = 2 * m.pairs;
    const int products = 2 + (m.splits > 1) + !poly.linear;           // arrivals of a step

    if (tid == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&bar.full[s], 2);
            mbar_init(&bar.peer_full[s], 1);
            mbar_init(&bar.empty[s], 2);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar.ready[i], WHOLE ? 2 : 1);                  // WHOLE: of both sums
            mbar_init(&bar.drained[i], 2 * (kWriters / 32));
        }
        mbar_init(&bar.mixed_ready, 1);
        mbar_init(&bar.mixed_drained, 2 * (kWriters / 32));
        mbar_init(&bar.done, 2);
        fence_mbar_init();
    }
    if (warp == kWriters / 32 + 2) tmem_alloc(&tmem_address, 512);
    tmem_fence_before();
    cluster.sync();
    tmem_fence_after();

    // For each product in turn: f(product, X's buffer, arrivals on the counter that its inputs need). Stops when f fails.
    // The threads that load and multiply stop, each for itself: nothing waits for them without a limit but the end. The
    // writers do not (write_product).
    auto each_product = [&](auto&& f) {
        for (int step = 0; step < steps; ++step) {
#pragma unroll 1                                                      // one copy of the code: three do not fit the instruction cache
            for (int p = GRAM; p <= STEP; ++p) {
                if (p == POLY && poly.linear) continue;
                if (!f(Product(p), step & 1, unsigned(step) * products + (p == GRAM ? 0 : p == POLY ? products - 2 : products - 1))) return false;
            }
        }
        return true;
    };

    if (tid == kWriters || tid == kWriters + 32) {
        const bool first = tid == kWriters;                           // the rows' operand, or the columns'
        unsigned k = 0, s = 0, phase = 1;                             // stages filled since the launch
        const bool ok = each_product([&](Product p, int from_x, unsigned before) {
            const int groups = first || w.wide(p) ? 2 : 1;
            const Planes from = first ? (p == GRAM ? w.x(from_x) : p == POLY ? w.gram : w.poly) : (p == POLY ? w.gram : w.x(from_x));
            const int units = w.units(p);
            for (int u = w.pair; u < units; u += w.pairs) {
                int ti, tj, k0, k1;
                w.unit(p, u, ti, tj, k0, k1);
                if (u == w.pair) {
                    if (!wait_counter(counter, before * ctas)) return false;
                    fence_proxy_async_all();
                }
                const int row = first ? ti * 4 + cta * 2 : (tj * 2 + cta) * groups;
                // of a symmetric matrix the 256 x 256 blocks above the diagonal are read across from below it
                const int below = p == GRAM ? k1 : !first && p == STEP ? -1 : ((first ? ti : tj * groups / 2) + 1) * 4;
                for (int kb = k0; kb < k1; ++kb, ++k) {
                    if (k >= kStages && !mbar_wait_bounded(&bar.empty[s], phase)) return false;
                    mbar_arrive_expect_tx(&bar.full[s], groups * kHalfBlock);
                    load_operand(stages + s * kStageBytes + (first ? 0 : kBlockBytes), from, row, groups, kb, kb >= below, &bar.full[s]);
                    if (++s == kStages) s = 0, phase ^= 1;
                }
                const Planes& added = p == POLY ? w.gram : w.x(from_x);
                for (int e = 0; e < w.extra(p); ++e, ++k) {
                    if (k >= kStages && !mbar_wait_bounded(&bar.empty[s], phase)) return false;
                    if (p == GRAM) {
                        mbar_arrive(&bar.full[s]);
                    } else {
                        const int block = tj * (w.wide(p) ? 4 : 2) + 2 * e + (first ? 0 : 1);
                        mbar_arrive_expect_tx(&bar.full[s], kBlockBytes);
                        bulk_copy_g2s(stages + s * kStageBytes + (first ? 0 : kBlockBytes),
                                      added.block(min(2 * ti + cta, added.row_blocks - 1), min(block, added.col_blocks - 1)), kBlockBytes, &bar.full[s]);
                    }
                    if (++s == kStages) s = 0, phase ^= 1;
                }
            }
            return true;
        });
        if (!ok) {
            // a stage that only the other operand's thread fills does not complete: wait for what was asked for here, with a limit
            *(volatile unsigned*)failed = 1;
            for (unsigned i = k > kStages ? k - kStages : 0; i < k; ++i) mbar_wait_bounded(&bar.full[i % kStages], (i / kStages) & 1);
        }
    } else if (tid == kWriters + 64 && cta == 1) {
        unsigned s = 0, phase = 0;
        const bool ok = each_product([&](Product p, int, unsigned) {
            for (int u = w.pair; u < w.units(p); u += w.pairs) {
                int ti, tj, k0, k1;
                w.unit(p, u, ti, tj, k0, k1);
                for (int kb = k0; kb < k1; ++kb) {
                    if (!mbar_wait_bounded(&bar.full[s], phase)) return false;
                    mbar_arrive_at(&bar.peer_full[s], 0);
                    if (++s == kStages) s = 0, phase ^= 1;
                }
                for (int e = 0; e < w.extra(p); ++e)
                    if (++s == kStages) s = 0, phase ^= 1;
            }
            return true;
        });
        if (!ok) *(volatile unsigned*)failed = 1;
        mbar_wait_bounded(&bar.done, 0);                              // no MMA reads this CTA when its memory is given up
    } else if ((tid == kWriters + 64 || tid == kWriters + 96) && cta == 0) {
        const bool mixed = tid == kWriters + 64;
        const uint32_t sums = mixed ? tmem_address + kMixedColumns : tmem_address;
        const int chunk_stages = m.chunk;
        unsigned s = 0, phase = 0, peer_phase = 0, tile = 0;          // peer_phase: one bit per stage
        unsigned used = 0, drained_phase = 0;                         // one bit per place of a chunk's sums
        const bool ok = each_product([&](Product p, int, unsigned) {
            const int groups_b = w.wide(p) ? 2 : 1;
            for (int u = w.pair; u < w.units(p); u += w.pairs, ++tile) {
                int ti, tj, k0, k1;
                w.unit(p, u, ti, tj, k0, k1);
                int of_chunk = 0;
                unsigned place = 0;
                const int below_a = p == GRAM ? k1 : (ti + 1) * 4, below_b = p == GRAM ? k1 : p == STEP ? -1 : (tj * groups_b / 2 + 1) * 4;
                for (int kb = k0; kb < k1; ++kb) {
                    const uint32_t a = smem_u32(stages + s * kStageBytes), bb = a + kBlockBytes;
                    const bool across_a = kb >= below_a, across_b = kb >= below_b;
                    const uint32_t instruction = f16_instruction(256, groups_b * 128, across_a, across_b);
                    const uint64_t a_hi = across_a ? mn_major_descriptor(a, kHalfBlock) : k_major_descriptor(a);
                    const uint64_t b_hi = across_b ? mn_major_descriptor(bb, kHalfBlock) : k_major_descriptor(bb);
                    const uint64_t step_a = (across_a ? mnMajorStep : kMajorStep) >> 4, step_b = (across_b ? mnMajorStep : kMajorStep) >> 4;
                    constexpr uint64_t lo = kPlaneOffset >> 4;
                    if (!mbar_wait_bounded(&bar.full[s], phase) || !mbar_wait_cluster(&bar.peer_full[s], (peer_phase >> s) & 1)) return false;
                    peer_phase ^= 1u << s;
                    // sums that are about to be overwritten are read
                    if (mixed) {
                        if (kb == k0 && tile > 0 && !mbar_wait_cluster(WHOLE ? &bar.drained[0] : &bar.mixed_drained, (tile - 1) & 1)) return false;
                    } else if (of_chunk == 0) {
                        if (!WHOLE && groups_b == 1 && kb > k0) place ^= 1;
                        if ((used >> place) & 1) {
                            if (!mbar_wait_cluster(&bar.drained[place], (drained_phase >> place) & 1)) return false;
                            drained_phase ^= 1u << place;
                        }
                        used |= 1u << place;
                    }
                    tmem_fence_after();
                    if (mixed) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {                 // 16 of the 64 in K
                            mma_f16(sums, a_hi + i * step_a, b_hi + i * step_b + lo, instruction, kb > k0 || i > 0);
                            mma_f16(sums, a_hi + i * step_a + lo, b_hi + i * step_b, instruction, true);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) mma_f16(sums + place * 128, a_hi + i * step_a, b_hi + i * step_b, instruction, of_chunk > 0 || i > 0);
                    }
                    mma_commit(&bar.empty[s]);
                    if (mixed) {
                        if (kb == k1 - 1) mma_commit(WHOLE ? &bar.ready[0] : &bar.mixed_ready);
                    } else if (of_chunk == chunk_stages - 1 || kb == k1 - 1) {
                        mma_commit(&bar.ready[place]);
                    }
                    if (++of_chunk == chunk_stages) of_chunk = 0;
                    if (++s == kStages) s = 0, phase ^= 1;
                }
                for (int e = 0; e < w.extra(p); ++e)
                    if (++s == kStages) s = 0, phase ^= 1;
            }
            return true;
        });
        if (!ok) *(volatile unsigned*)failed = 1;
        mma_commit(&bar.done);
        mbar_wait_bounded(&bar.done, 0);                              // nothing in flight when the TMEM is freed
    } else if (warp < kWriters / 32) {
        WriterCounts n = {0, 0, 0};
        // This CTA's part of a product is written: by bulk copies, for which the lanes that issued them wait, or by all threads
        // with plain stores. Others read it by bulk copies.
        auto arrive = [&](bool plain) {
            if ((tid & 31) == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
            if (plain) __threadfence();
            if (plain || (tid & 31) == 0) fence_proxy_async_all();
            writers_sync();
            if (tid == 0) asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(counter) : "memory");
        };
        auto wait = [&](unsigned arrivals) {                          // the warp goes on when its first lane has seen the counter
            bool ok = true;
            if ((tid & 31) == 0) ok = wait_counter(counter, arrivals * ctas);
            return to_warp(ok);
        };
        const uint32_t tmem = tmem_address;
        bool ok = int(blockIdx.x) * (kWriters / 32) + warp != b.lost_wait;
        if (!ok && (tid & 31) == 0) report_check(CHECK_MBARRIER_TIMEOUT);
        each_product([&](Product p, int from_x, unsigned before) {
            // a pair without tiles in a product must not arrive for the next one early: the counter has no names
            ok = ok && wait(before);
            const Planes& to = p == STEP ? w.x(from_x ^ 1) : p == POLY || poly.linear ? w.poly : w.gram;
            const float c0 = p == STEP ? poly.step_from : p == POLY ? poly.poly_from : 0.f;
            const float c1 = p == STEP ? poly.step_factor : p == POLY ? poly.poly_factor : poly.gram_factor;
            write_product<WHOLE>(p, w, bar, stages, tmem, cta, n, to, c0, c1, m.chunk, partial, ok);
            if (p == GRAM && w.splits > 1) {
                arrive(true);
                ok = ok && wait(before + 1);
                reduce_gram(w, cta, partial, to, c1);
            }
            arrive(p == GRAM && w.splits > 1);
            return true;
        });
        if (!ok) *(volatile unsigned*)failed = 1;
        tmem_fence_before();
    }
    __syncwarp();
    cluster.sync();                                                   // the pair's memory and barriers are used until here
    if (warp == kWriters / 32 + 2) {
        tmem_fence_after();
        tmem_free(tmem_address, 512);
    }
}

// ---- matrices with a short side: the whole chain in one launch, fp32 -------------------------------------------------
// One cluster per matrix. Each CTA keeps X for its share of the columns in shared memory over all steps; per step every CTA
// adds up all shares of X X^T over distributed shared memory, forms P = a I + b A + c A A for itself and multiplies its own
// columns with it in place. Nothing goes through global memory between the update's elements and the result, and the products
// are fp32. Up to 16 rows; above, the shared memory's bandwidth binds (64 x 160: 49 us in this form, 41 on the tensor cores).
// What bounds it is the chain of latencies, five barriers a step: 16 x 40 takes 13 us, 16 x 2000 (eight CTAs) 20 us.
constexpr int kShortThreads = 512;
constexpr int kShortWarps = kShortThreads / 32;
constexpr int kShortRows = 16;
struct ClusterBatch {
    Matrix m[kMaxMatrices];
};
// Sizes for X padded to MP = 8 or 16 rows: 4 x 4 tiles on and below the diagonal of X X^T.
__host__ __device__ constexpr int short_padded_rows(int rows) { return rows <= 8 ? 8 : 16; }
__host__ __device__ constexpr int short_tiles(int mp) { return (mp / 4) * (mp / 4 + 1) / 2; }
__host__ __device__ constexpr int short_packed(int mp) { return short_tiles(mp) * 16; }
__host__ __device__ constexpr int short_columns(int cols, int ranks) { return ((cols + ranks - 1) / ranks + 3) & ~3; }
__host__ __device__ constexpr int short_pitch(int columns) { return ((columns + 27) / 32) * 32 + 4; }    // = 4 mod 32 banks, >= columns
__host__ __device__ constexpr size_t short_smem(int rows, int cols, int ranks) {
    const int mp = short_padded_rows(rows);
    return size_t(mp * short_pitch(short_columns(cols, ranks)) + 2 * mp * (mp + 4) + 2 * short_packed(mp)) * sizeof(float);
}

// Sums 16 values over the warp's lanes; returns the sum of value lane / 2 (both lanes of a pair hold it).
__device__ __forceinline__ float warp_sum16(const float (&v)[16], int lane) {
    float a[8], b[4], c[2];
    const bool h16 = lane & 16, h8 = lane & 8, h4 = lane & 4, h2 = lane & 2;
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = (h16 ? v[8 + i] : v[i]) + __shfl_xor_sync(0xffffffffu, h16 ? v[i] : v[8 + i], 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = (h8 ? a[4 + i] : a[i]) + __shfl_xor_sync(0xffffffffu, h8 ? a[i] : a[4 + i], 8);
#pragma unroll
    for (int i = 0; i < 2; ++i) c[i] = (h4 ? b[2 + i] : b[i]) + __shfl_xor_sync(0xffffffffu, h4 ? b[i] : b[2 + i], 4);
    const float d = (h2 ? c[1] : c[0]) + __shfl_xor_sync(0xffffffffu, h2 ? c[0] : c[1], 2);
    return d + __shfl_xor_sync(0xffffffffu, d, 1);
}

// acc[4 i + j] += row (pi + i down) . row (pj + j down) over c = first, first + step, .. < length, four columns at a time
__device__ __forceinline__ void tile_product(float (&acc)[16], const float* pi, const float* pj, int down, int first, int step, int length) {
    for (int c = first; c < length; c += step) {
        float4 p[4], q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            p[i] = *reinterpret_cast<const float4*>(pi + i * down + c);
            q[i] = *reinterpret_cast<const float4*>(pj + i * down + c);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                acc[4 * i + j] += p[i].x * q[j].x;
                acc[4 * i + j] += p[i].y * q[j].y;
                acc[4 * i + j] += p[i].z * q[j].z;
                acc[4 * i + j] += p[i].w * q[j].w;
            }
    }
}

// Tile number -> (row, column) of the tile on or below the diagonal.
__device__ __forceinline__ void tile_place(int tile, int& ti, int& tj) {
    ti = 0;
    while ((ti + 1) * (ti + 2) / 2 <= tile) ++ti;
    tj = tile - ti * (ti + 1) / 2;
}

// X X^T packed: element (4 i + j) of tile t at (4 i + j) * tiles + t. Tile (ti, tj) holds rows ti + side i and columns
// tj + side j, so that neighbouring tiles read neighbouring rows, which the pitch puts into different banks.
// A warp per tile, its lanes share the columns. done(e, value) is called once for every packed element.
template <int MP, typename Done>
__device__ __forceinline__ void symmetric_product(const float* from, int pitch, int length, Done&& done) {
    constexpr int side = MP / 4, tiles = short_tiles(MP);
    static_assert(tiles <= kShortWarps, "a warp per tile");
    const int lane = threadIdx.x & 31, tile = threadIdx.x >> 5;
    if (tile < tiles) {
        int ti, tj;
        tile_place(tile, ti, tj);
        float acc[16] = {};
        tile_product(acc, from + ti * pitch, from + tj * pitch, side * pitch, lane * 4, 128, length);
        const float v = warp_sum16(acc, lane);
        if ((lane & 1) == 0) done((lane >> 1) * tiles + tile, v);
    }
}
// Packed element -> its places (row, column) and (column, row) in a matrix of the given pitch.
template <int MP>
__device__ __forceinline__ void packed_places(int e, int pitch, int& at, int& mirror) {
    constexpr int side = MP / 4, tiles = short_tiles(MP);
    int ti, tj;
    tile_place(e % tiles, ti, tj);
    const int i = e / tiles, r = ti + side * (i >> 2), c = tj + side * (i & 3);
    at = r * pitch + c;
    mirror = c * pitch + r;
}

// X <- P X in place, RT x 4 elements per thread: a warp holds all rows of its columns, so what it overwrites it alone reads.
template <int MP, int RT>
__device__ __forceinline__ void multiply_in_place(float* x, int pitch, int columns, const float* p) {
    constexpr int gp = MP + 4, row_tiles = MP / RT, col_tiles = 32 / row_tiles;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row = (lane % row_tiles) * 4, my_col = (lane / row_tiles) * 4;
    for (int c0 = warp * col_tiles * 4; c0 < columns; c0 += kShortWarps * col_tiles * 4) {
        const int c = c0 + my_col;
        const bool in = c < columns;
        float acc[RT][4] = {};
        if (in) {
            const float* xc = x + c;
            const float* pr = p + row;
#pragma unroll 8
            for (int k = 0; k < MP; ++k) {
                const float4 v = *reinterpret_cast<const float4*>(xc + k * pitch);
#pragma unroll
                for (int h = 0; h < RT / 4; ++h) {
                    const float4 q4 = *reinterpret_cast<const float4*>(pr + k * gp + h * row_tiles * 4);
                    const float q[4] = {q4.x, q4.y, q4.z, q4.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        acc[h * 4 + i][0] += q[i] * v.x, acc[h * 4 + i][1] += q[i] * v.y;
                        acc[h * 4 + i][2] += q[i] * v.z, acc[h * 4 + i][3] += q[i] * v.w;
                    }
                }
            }
        }
        __syncwarp();
        if (in)
#pragma unroll
            for (int i = 0; i < RT; ++i)
                *reinterpret_cast<float4*>(x + (row + (i / 4) * row_tiles * 4 + (i & 3)) * pitch + c) =
                    make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
    }
}

template <typename T, bool MUON, int MP>
__device__ __forceinline__ void short_matrix(const Matrix& m, int ranks, int rank, const Momentum& mo, int steps, float ca, float cb, float cc,
                                             float epsilon, float* smem, double* warp_sum, double* cta_sum) {
    constexpr int gp = MP + 4, packed = short_packed(MP);
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const bool tall = m.rows > m.cols;
    const int wide_rows = tall ? m.cols : m.rows, wide_cols = tall ? m.rows : m.cols;
    const int columns = short_columns(wide_cols, ranks), pitch = short_pitch(columns);
    const int col0 = rank * columns, here = max(0, min(columns, wide_cols - col0));
    float* x = smem;
    float* gram = x + MP * pitch;                // A
    float* poly = gram + MP * gp;                // P = a I + b A + c A A
    float* share = poly + MP * gp;               // the CTA's share of A, packed; two buffers in turn

    for (int i = tid * 4; i < MP * pitch; i += kShortThreads * 4) *reinterpret_cast<float4*>(x + i) = make_float4(0.f, 0.f, 0.f, 0.f);
    __syncthreads();
    // neighbouring threads along the rows of the update: `inner` elements of `outer` rows
    const int inner = tall ? wide_rows : here, outer = inner > 0 ? (tall ? here : wide_rows) : 0;
    const int step_outer = inner > 0 ? kShortThreads / inner : 0, step_inner = inner > 0 ? kShortThreads % inner : 0;
    const long long first = tall ? 0 : col0, first_row = tall ? col0 : 0;
    const int start_outer = inner > 0 ? tid / inner : 0, start_inner = inner > 0 ? tid % inner : 0;
    auto next = [&](int& o, int& i) {
        o += step_outer;
        i += step_inner;
        if (i >= inner) i -= inner, ++o;
    };
    constexpr int kBatch = 8;                                         // loads in flight per thread
    double s = 0.;
    for (int o0 = start_outer, i0 = start_inner; o0 < outer;) {
        float u[kBatch], old[kBatch];
        int o = o0, i = i0;
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const bool in = o < outer;
            u[j] = in ? float(static_cast<const T*>(m.update)[(first_row + o) * m.update_stride + first + i]) : 0.f;
            if constexpr (MUON) old[j] = in ? m.momentum[(first_row + o) * m.cols + first + i] : 0.f;
            next(o, i);
        }
        o = o0, i = i0;
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            if (o < outer) {
                if constexpr (MUON) {
                    const float now = mo.beta * old[j] + mo.one_minus_beta * u[j];
                    m.momentum[(first_row + o) * m.cols + first + i] = now;
                    u[j] = mo.nesterov ? mo.one_minus_beta * u[j] + mo.beta * now : now;
                }
                x[tall ? i * pitch + o : o * pitch + i] = u[j];
                s += double(u[j]) * double(u[j]);
            }
            next(o, i);
        }
        o0 = o, i0 = i;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) warp_sum[warp] = s;
    __syncthreads();
    s = lane < kShortWarps ? warp_sum[lane] : 0.;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    s = __shfl_sync(0xffffffffu, s, 0);
    if (ranks > 1) {
        if (tid == 0) *cta_sum = s;
        cluster.sync();
        s = lane < ranks ? *cluster.map_shared_rank(cta_sum, lane) : 0.;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        s = __shfl_sync(0xffffffffu, s, 0);
    }
    // 1 / norm is no normal fp32 number for norms above 2^126: X is made smaller by a power of two first
    const double norm = sqrt(s) + double(epsilon);
    const float before = norm > 0x1p100 ? 0x1p-100f : 1.f, factor = float(1. / (norm * double(before)));
    for (int i = tid * 4; i < MP * pitch; i += kShortThreads * 4) {
        float4 v = *reinterpret_cast<float4*>(x + i);
        v.x = v.x * before * factor, v.y = v.y * before * factor, v.z = v.z * before * factor, v.w = v.w * before * factor;
        *reinterpret_cast<float4*>(x + i) = v;
    }
    // where this thread's element of the packed sums goes (the same in every step)
    static_assert(packed <= kShortThreads, "one element per thread");
    const bool has = tid < packed;
    int at = 0, mirror = 0;
    if (has) packed_places<MP>(tid, gp, at, mirror);
    __syncthreads();

    for (int step = 0; step < steps; ++step) {
        // A: every CTA adds up all shares in their order. A share's buffer is written again two steps, so one barrier, later.
        float* mine = share + (step & 1) * packed;
        symmetric_product<MP>(x, pitch, columns, [&](int e, float v) { mine[e] = v; });
        if (ranks > 1) cluster.sync();
        else __syncthreads();
        if (has) {
            float v = 0.f;
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (q < ranks) v += (ranks > 1 ? cluster.map_shared_rank(mine, q) : mine)[tid];
            gram[at] = gram[mirror] = v;
        }
        __syncthreads();
        symmetric_product<MP>(gram, gp, MP, [&](int e, float v) {
            int a, b;
            packed_places<MP>(e, gp, a, b);
            poly[a] = poly[b] = cb * gram[a] + cc * v + (a == b ? ca : 0.f);
        });
        __syncthreads();
        // the taller tile reads less per product, the lower one has more warps at work while there are few columns
        if (columns * MP >= 4 * 4 * kShortThreads) multiply_in_place<MP, 8>(x, pitch, columns, poly);
        else multiply_in_place<MP, 4>(x, pitch, columns, poly);
        __syncthreads();
    }
    T* out = static_cast<T*>(m.out);
#pragma unroll 4
    for (int o = start_outer, i = start_inner; o < outer; next(o, i)) {
        T* to = out + (first_row + o) * m.out_stride + first + i;
        const float v = x[tall ? i * pitch + o : o * pitch + i];
        *to = T(MUON ? float(*to) * mo.decay - m.rate * v : v);
    }
    if (ranks > 1) cluster.sync();                                    // no CTA leaves while its shared memory is read
}

// ---- matrices with a side of 17 to 128: the whole chain in one launch, on the tensor cores ---------------------------
// One cluster per matrix; each CTA keeps X for its share of the columns in shared memory, as the chain's planes (blocks of MP
// rows x 64 columns). Per step: X X^T of the CTA's columns; the shares are added up over distributed shared memory, CTA q
// summing rows q MP / ranks .. and handing them to all as planes; B = b A + c A A in A's place, each CTA for itself;
// X <- a X + B X in place. All accumulators are in tensor memory; additions per accumulator are few (128 in K), so that the
// losses of the module comment stay small. What bounds it is the chain of latencies, about eight barriers a step: 64 x 160 takes 40 us, 0.28
// TFLOP/s of the polynomial's. The update is held in registers over the norm, and of 128 a thread (512 threads fill the register
// file) 236 to 252 bytes spill; what that costs is not known.
constexpr int kMidThreads = 512;
constexpr int kMidWarps = kMidThreads / 32;
__host__ __device__ constexpr int mid_rows(int rows) { return rows <= 64 ? 64 : 128; }
__host__ __device__ constexpr int mid_max_blocks(int mp) { return mp == 64 ? 8 : 3; }                    // of 64 columns per CTA
__host__ __device__ constexpr int mid_block_bytes(int mp) { return mp * 64 * 4; }
__host__ __device__ constexpr int mid_blocks(int cols, int ranks) { return ((cols + ranks - 1) / ranks + 63) / 64; }
__host__ __device__ constexpr int mid_smem(int mp, int blocks) { return blocks * mid_block_bytes(mp) + 2 * mp * mp * 4 + 1024; }

template <typename T, bool MUON, int MP>
__device__ __forceinline__ void mid_matrix(const Matrix& m, int ranks, int rank, const Momentum& mo, int steps, const Polynomial& poly, float epsilon,
                                           uint8_t* smem, uint32_t tmem, uint64_t* bar, double* warp_sum, double* cta_sum) {
    constexpr int kBlock = mid_block_bytes(MP), kMaxUnits = MP * mid_max_blocks(MP) * 8 / kMidThreads;
    constexpr int kPerSum = MP == 64 ? 2 : 1;                         // blocks of X X^T per accumulator
    constexpr uint32_t kMixedGram = 512 - MP;
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const bool tall = m.rows > m.cols;
    const int wide_rows = tall ? m.cols : m.rows, wide_cols = tall ? m.rows : m.cols;
    const int blocks = mid_blocks(wide_cols, ranks), col0 = rank * blocks * 64;
    uint8_t* x = smem;
    uint8_t* gram = x + blocks * kBlock;                              // A's planes, then B's
    float* share = reinterpret_cast<float*>(gram + MP * MP * 4);      // the CTA's part of A; float4 c of row r at c ^ (r & 7)
    bool ok = true;
    unsigned phase = 0;
    auto wait_mma = [&]() {
        ok = warp_wait(bar, phase) && ok;
        phase ^= 1;
        tmem_fence_after();
    };

    // the update: units of eight columns of a row, neighbouring threads along the rows of the update
    float u[kMaxUnits][8];
    double s = 0.;
    const int units = MP * blocks * 8, row_units = blocks * 8;
    const unsigned reciprocal = 0xffffffffu / unsigned(row_units) + 1u;                // exact quotients of numbers below 4096
    const T* update = static_cast<const T*>(m.update);
    const bool vectors = !tall && rows_aligned(update, m.update_stride, sizeof(T)), momentum_vectors = !tall && rows_aligned(m.momentum, m.cols, 4);
    auto place = [&](int unit, int& row, int& col) {                                   // in the wide form
        row = tall ? unit & (MP - 1) : int(__umulhi(unsigned(unit), reciprocal));
        col = col0 + (tall ? unit / MP : unit - row * row_units) * 8;
    };
#pragma unroll
    for (int i = 0; i < kMaxUnits; ++i) {
        int row, col;
        place(tid + i * kMidThreads, row, col);
        const bool in = tid + i * kMidThreads < units && row < wide_rows;
        float old[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) u[i][e] = old[e] = 0.f;
        if (in && !tall && col + 8 <= wide_cols) {
            load8(update + row * m.update_stride + col, vectors, u[i]);
            if constexpr (MUON) load8(m.momentum + (long long)row * m.cols + col, momentum_vectors, old);
        } else if (in) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (col + e < wide_cols) {
                    const long long rr = tall ? col + e : row, cc = tall ? row : col + e;
                    u[i][e] = float(update[rr * m.update_stride + cc]);
                    if constexpr (MUON) old[e] = m.momentum[rr * m.cols + cc];
                }
            }
        }
        if constexpr (MUON) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                old[e] = mo.beta * old[e] + mo.one_minus_beta * u[i][e];
                u[i][e] = mo.nesterov ? mo.one_minus_beta * u[i][e] + mo.beta * old[e] : old[e];
            }
            if (in && !tall && col + 8 <= wide_cols) {
                store8(m.momentum + (long long)row * m.cols + col, momentum_vectors, old);
            } else if (in) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (col + e < wide_cols) m.momentum[tall ? (long long)(col + e) * m.cols + row : (long long)row * m.cols + col + e] = old[e];
            }
        }
    }
#pragma unroll
    for (int i = 0; i < kMaxUnits; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) s += double(u[i][e]) * double(u[i][e]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) warp_sum[warp] = s;
    __syncthreads();
    s = lane < kMidWarps ? warp_sum[lane] : 0.;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    s = __shfl_sync(0xffffffffu, s, 0);
    if (ranks > 1) {
        if (tid == 0) *cta_sum = s;
        cluster.sync();
        s = lane < ranks ? *cluster.map_shared_rank(cta_sum, lane) : 0.;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        s = __shfl_sync(0xffffffffu, s, 0);
    }
    const float factor = float(double(kScaleX) / (sqrt(s) + double(epsilon)));
    const uint4 none = {};
#pragma unroll
    for (int i = 0; i < kMaxUnits; ++i) {
        int row, col;
        place(tid + i * kMidThreads, row, col);
        if (tid + i * kMidThreads < units) {
            const int chunk = (col - col0) >> 3;
            uint4 hi, lo;
            split8<false>(u[i], factor, 0.f, none, none, hi, lo);
            uint8_t* at = x + (chunk >> 3) * kBlock + swizzled_offset(row, chunk & 7);
            *reinterpret_cast<uint4*>(at) = hi;
            *reinterpret_cast<uint4*>(at + kPlaneOffset) = lo;
        }
    }
    fence_proxy_async();
    __syncthreads();

    const int quarter = warp & 3, part = warp >> 2, row = quarter * 32 + lane;         // rows of the warp, share of the columns
    const bool rows_here = quarter * 32 < MP;
    const uint32_t lanes = uint32_t(quarter * 32) << 16;
    constexpr uint64_t lo_plane = kPlaneOffset >> 4;
    const uint32_t x_at = smem_u32(x), gram_at = smem_u32(gram);
    const int last = min(blocks * 64, wide_cols - col0);              // columns of this CTA that hold something
    // two threads issue: the mixed products and hi hi (80 cycles for each MMA that a thread issues)
    const bool issues_mixed = tid == 0, issues_main = tid == 32;
    for (int step = 0; step < steps; ++step) {
        const int sums = (blocks + kPerSum - 1) / kPerSum;
        if (issues_mixed || issues_main) {
            tmem_fence_after();
            constexpr uint32_t instruction = f16_instruction(128, MP, false, false);
            uint64_t a = k_major_descriptor(x_at);
            uint32_t sum = tmem;
            bool more = false;                                        // the accumulator holds something already
            for (int k = 0; k * 16 < last || k == 0; ++k) {
                if (issues_mixed) {
                    mma_f16_single(tmem + kMixedGram, a, a + lo_plane, instruction, k > 0);
                    mma_f16_single(tmem + kMixedGram, a + lo_plane, a, instruction, true);
                } else {
                    mma_f16_single(sum, a, a, instruction, more);
                }
                a += (k & 3) == 3 ? (kBlock - 3 * kMajorStep) >> 4 : kMajorStep >> 4;
                more = (k + 1) % (4 * kPerSum) != 0;
                if (!more) sum += MP;
            }
            mma_commit_single(bar);
        }
        wait_mma();
        if (rows_here) {
#pragma unroll 1
            for (int q = part * 32; q < MP; q += (kMidWarps / 4) * 32) {
                float v[32], add[32];
                tmem_load32(tmem + lanes + kMixedGram + q, v, tmem + lanes + q, add);
                for (int i = 0;;) {
                    const float loss = 0x1p-25f * 4.f * float(min(kPerSum, blocks - i * kPerSum));
#pragma unroll
                    for (int e = 0; e < 32; ++e) v[e] += add[e] * (q + e == row ? 1.f + 2.f * loss : 1.f + 0.7f * loss);
                    if (++i >= sums || i * kPerSum * 64 >= last) break;                // no columns, no sums
                    tmem_load32(tmem + lanes + i * MP + q, add);
                }
                if (ranks > 1) {
                    float4* to = reinterpret_cast<float4*>(share) + row * (MP / 4);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        to[(q / 4 + e) ^ (row & 7)] = make_float4(v[4 * e] * poly.gram_factor, v[4 * e + 1] * poly.gram_factor,
                                                                  v[4 * e + 2] * poly.gram_factor, v[4 * e + 3] * poly.gram_factor);
                } else {
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        uint4 hi, lo;
                        split8<false>(v + g * 8, poly.gram_factor, 0.f, none, none, hi, lo);
                        uint8_t* at = gram + (q >> 6) * kBlock + swizzled_offset(row, ((q & 63) >> 3) + g);
                        *reinterpret_cast<uint4*>(at) = hi;
                        *reinterpret_cast<uint4*>(at + kPlaneOffset) = lo;
                    }
                }
            }
        }
        tmem_fence_before();
        if (ranks > 1) {
            cluster.sync();
            const int each = MP / ranks;                              // rows that this CTA sums
            for (int i = tid; i < each * (MP / 8); i += kMidThreads) {
                const int r = rank * each + i / (MP / 8), chunk = i % (MP / 8);
                float4 a[8], b[8];
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    if (q < ranks) {
                        const float4* from = reinterpret_cast<const float4*>(cluster.map_shared_rank(share, q)) + r * (MP / 4);
                        a[q] = from[(2 * chunk) ^ (r & 7)];
                        b[q] = from[(2 * chunk + 1) ^ (r & 7)];
                    }
                }
                float v[8] = {};
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (q < ranks)
                        v[0] += a[q].x, v[1] += a[q].y, v[2] += a[q].z, v[3] += a[q].w, v[4] += b[q].x, v[5] += b[q].y, v[6] += b[q].z, v[7] += b[q].w;
                uint4 hi, lo;
                split8<false>(v, 1.f, 0.f, none, none, hi, lo);
                const uint32_t at = (chunk >> 3) * kBlock + swizzled_offset(r, chunk & 7);
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    if (q < ranks) {
                        uint8_t* to = cluster.map_shared_rank(gram, q) + at;
                        *reinterpret_cast<uint4*>(to) = hi;
                        *reinterpret_cast<uint4*>(to + kPlaneOffset) = lo;
                    }
                }
            }
            fence_proxy_async_all();
            cluster.sync();
            if (issues_mixed || issues_main) fence_proxy_async_all();
        } else {
            fence_proxy_async();
            __syncthreads();
        }
        if (!poly.linear) {
            if (issues_mixed || issues_main) {
                tmem_fence_after();
                constexpr uint32_t instruction = f16_instruction(128, MP, false, false);
#pragma unroll
                for (int k = 0; k < MP / 16; ++k) {
                    const uint64_t a = k_major_descriptor(gram_at + (k >> 2) * kBlock + (k & 3) * kMajorStep);
                    if (issues_mixed) {
                        mma_f16_single(tmem + MP, a, a + lo_plane, instruction, k > 0);
                        mma_f16_single(tmem + MP, a + lo_plane, a, instruction, true);
                    } else {
                        mma_f16_single(tmem, a, a, instruction, k > 0);
                    }
                }
                mma_commit_single(bar);
            }
            wait_mma();
            if (rows_here) {
                constexpr float loss = 0x1p-25f * float(MP / 16);
#pragma unroll 1
                for (int q = part * 32; q < MP; q += (kMidWarps / 4) * 32) {
                    float v[32], add[32];
                    tmem_load32(tmem + lanes + MP + q, v, tmem + lanes + q, add);
#pragma unroll
                    for (int e = 0; e < 32; ++e) v[e] += add[e] * (q + e == row ? 1.f + 2.4f * loss : 1.f + 0.7f * loss);
                    uint8_t* block = gram + (q >> 6) * kBlock;
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        uint8_t* at = block + swizzled_offset(row, ((q & 63) >> 3) + g);
                        const uint4 in_hi = *reinterpret_cast<const uint4*>(at), in_lo = *reinterpret_cast<const uint4*>(at + kPlaneOffset);
                        uint4 hi, lo;
                        split8<true>(v + g * 8, poly.poly_factor, poly.poly_from, in_hi, in_lo, hi, lo);
                        *reinterpret_cast<uint4*>(at) = hi;
                        *reinterpret_cast<uint4*>(at + kPlaneOffset) = lo;
                    }
                }
            }
            fence_proxy_async();
            tmem_fence_before();
            __syncthreads();
        }
        // 256 columns at a time: 256 of tensor memory for each of the two sums
        for (int c0 = 0; c0 < last; c0 += 256) {
            const int n = min(256, (last - c0 + 15) & ~15);
            if (issues_mixed || issues_main) {
                tmem_fence_after();
                const uint32_t instruction = f16_instruction(128, n, false, true);
#pragma unroll
                for (int k = 0; k < MP / 16; ++k) {
                    const uint64_t a = k_major_descriptor(gram_at + (k >> 2) * kBlock + (k & 3) * kMajorStep);
                    const uint64_t b = mn_major_descriptor(x_at + (c0 >> 6) * kBlock + k * mnMajorStep, kBlock);
                    if (issues_mixed) {
                        mma_f16_single(tmem + 256, a, b + lo_plane, instruction, k > 0);
                        mma_f16_single(tmem + 256, a + lo_plane, b, instruction, true);
                    } else {
                        mma_f16_single(tmem, a, b, instruction, k > 0);
                    }
                }
                mma_commit_single(bar);
            }
            wait_mma();
            if (rows_here) {
                constexpr float made_good = 1.f + 0.7f * 0x1p-25f * float(MP / 16);
#pragma unroll 1
                for (int q = part * 32; q < n; q += (kMidWarps / 4) * 32) {
                    float v[32], add[32];
                    tmem_load32(tmem + lanes + 256 + q, v, tmem + lanes + q, add);
#pragma unroll
                    for (int e = 0; e < 32; ++e) v[e] += add[e] * made_good;
                    uint8_t* block = x + ((c0 + q) >> 6) * kBlock;
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        // beyond n the sums are not this product's; nothing is stored there but zeros
                        if (q + g * 8 < n) {
                            uint8_t* at = block + swizzled_offset(row, ((q & 63) >> 3) + g);
                            const uint4 in_hi = *reinterpret_cast<const uint4*>(at), in_lo = *reinterpret_cast<const uint4*>(at + kPlaneOffset);
                            uint4 hi, lo;
                            split8<true>(v + g * 8, poly.step_factor, poly.step_from, in_hi, in_lo, hi, lo);
                            *reinterpret_cast<uint4*>(at) = hi;
                            *reinterpret_cast<uint4*>(at + kPlaneOffset) = lo;
                        }
                    }
                }
            }
            fence_proxy_async();
            tmem_fence_before();
            __syncthreads();
        }
    }
    if (!ok) report_check(CHECK_MBARRIER_TIMEOUT);
    T* out = static_cast<T*>(m.out);
    const bool out_vectors = !tall && rows_aligned(out, m.out_stride, sizeof(T));
#pragma unroll 2
    for (int unit = tid; unit < units; unit += kMidThreads) {
        int r, col;
        place(unit, r, col);
        if (r >= wide_rows || col >= wide_cols) continue;
        const int chunk = (col - col0) >> 3;
        const uint8_t* at = x + (chunk >> 3) * kBlock + swizzled_offset(r, chunk & 7);
        Chunk hi, lo;
        hi.raw = *reinterpret_cast<const uint4*>(at);
        lo.raw = *reinterpret_cast<const uint4*>(at + kPlaneOffset);
        float v[8], old[8];
        const bool whole = !tall && col + 8 <= wide_cols;
        if (MUON && whole) load8(out + r * m.out_stride + col, out_vectors, old);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[e] = (__half2float(hi.h[e]) + __half2float(lo.h[e])) * (1.f / kScaleX);
            if (!ok) v[e] = __int_as_float(0x7fffffff);
            if (MUON && whole) v[e] = old[e] * mo.decay - m.rate * v[e];
        }
        if (whole) {
            store8(out + r * m.out_stride + col, out_vectors, v);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (col + e < wide_cols) {
                    T* to = out + (tall ? (col + e) * m.out_stride + r : r * m.out_stride + col + e);
                    *to = T(MUON ? float(*to) * mo.decay - m.rate * v[e] : v[e]);
                }
            }
        }
    }
    if (ranks > 1) cluster.sync();                                    // no CTA leaves while its shared memory is read or written
}

// One cluster per matrix, of either kind, or without the code for the shortest ones (64 x 160: 41 us instead of 45).
template <typename T, bool MUON, bool SHORT>
__global__ void __launch_bounds__(kMidThreads, 1) cluster_kernel(const __grid_constant__ ClusterBatch b, int ranks, Momentum mo, int steps, float ca,
                                                                 float cb, float cc, Polynomial poly, float epsilon) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ double warp_sum[kMidWarps], cta_sum;
    __shared__ uint64_t bar;
    __shared__ uint32_t tmem_address;
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const Matrix& m = b.m[blockIdx.x / unsigned(ranks)];
    const int rank = int(blockIdx.x % unsigned(ranks)), rows = min(m.rows, m.cols);
    if (SHORT && rows <= kShortRows) {
        float* floats = reinterpret_cast<float*>(smem);
        if (rows <= 8) short_matrix<T, MUON, 8>(m, ranks, rank, mo, steps, ca, cb, cc, epsilon, floats, warp_sum, &cta_sum);
        else short_matrix<T, MUON, 16>(m, ranks, rank, mo, steps, ca, cb, cc, epsilon, floats, warp_sum, &cta_sum);
        return;
    }
    if (threadIdx.x == 0) {
        mbar_init(&bar, 2);                                           // commits of the two issuing threads
        fence_mbar_init();
    }
    if (threadIdx.x < 32) tmem_alloc_single(&tmem_address, 512);
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = tmem_address;
    if (rows <= 64) mid_matrix<T, MUON, 64>(m, ranks, rank, mo, steps, poly, epsilon, smem, tmem, &bar, warp_sum, &cta_sum);
    else mid_matrix<T, MUON, 128>(m, ranks, rank, mo, steps, poly, epsilon, smem, tmem, &bar, warp_sum, &cta_sum);
    __syncthreads();
    if (threadIdx.x < 32) tmem_free_single(tmem, 512);
}

// ---- host side -------------------------------------------------------------------------------------------------------
int ceil_div(long long a, long long b) { return int((a + b - 1) / b); }

// Cycles of a product with a number of pairs, for the choice of tiles and pairs: measured per 64 in K 1520 cycles at 256
// columns (the MMAs' own time is 1536) and 1440 at 128 (the barriers' latencies, behind the operands' traffic in shared
// memory); a tile costs about 8000 and 6000 more to start and to write, and a wide one 1400 for each further chunk.
long long product_cycles(long long tiles, int wide, long long k_blocks, int pairs, int chunk) {
    return (tiles + pairs - 1) / pairs * (wide ? 1520 * k_blocks + 8000 + (k_blocks - 1) / chunk * 1400 : 1440 * k_blocks + 6000);
}
long long step_tiles(const Matrix& m, int wide) { return (long long)((m.row_tiles + 1) / 2) * ((m.col_blocks + (wide ? 3 : 1)) / (wide ? 4 : 2)); }

// Chooses tile widths and shares of the columns for a matrix with some pairs; returns the step's cycles.
long long plan(Matrix& m, int pairs) {
    const long long barrier = 8000;
    long long total = 2 * barrier, best = -1;
    m.pairs = pairs;
    for (int wide = 0; wide < 2; ++wide) {
        const long long tiles = symmetric_tiles(m.row_tiles, wide);
        for (int splits = 1; splits <= 32; splits *= 2) {
            if (splits > 1 && (tiles * splits > pairs || m.col_blocks < 4 * splits)) break;
            const long long reduce = splits > 1 ? 22000 + 400 * splits * ((tiles * (wide ? 64 : 32) + pairs * 16 - 1) / (pairs * 16)) : 0;
            const long long t = product_cycles(tiles * splits, wide, m.col_blocks / splits, pairs, m.chunk) + reduce;
            if (best < 0 || t < best) best = t, m.gram_wide = wide, m.splits = splits;
        }
    }
    total += best;
    const long long p0 = product_cycles(symmetric_tiles(m.row_tiles, 0), 0, 2 * m.row_tiles, pairs, m.chunk);
    const long long p1 = product_cycles(symmetric_tiles(m.row_tiles, 1), 1, 2 * m.row_tiles, pairs, m.chunk);
    m.poly_wide = p1 <= p0;
    const long long s0 = product_cycles(step_tiles(m, 0), 0, 2 * m.row_tiles, pairs, m.chunk), s1 = product_cycles(step_tiles(m, 1), 1, 2 * m.row_tiles, pairs, m.chunk);
    m.step_wide = s1 <= s0;
    return total + (p1 <= p0 ? p1 : p0) + (s1 <= s0 ? s1 : s0) + barrier;
}

// Pairs beyond this have nothing to do.
long long most_units(const Matrix& m) {
    const long long gram = (long long)symmetric_tiles(m.row_tiles, 0) * (m.col_blocks / 4 > 1 ? m.col_blocks / 4 : 1);
    const long long step = step_tiles(m, 0);
    return gram > step ? gram : step;
}

// Stages of the longest sum among a matrix's products.
int longest_sum(const Matrix& m) { return std::max(2 * m.row_tiles, ceil_div(m.col_blocks, m.splits)); }

// Hands out `pairs` CTA pairs: one each, the others to whoever takes longest.
void hand_out(Batch& b, int pairs) {
    long long cycles[kMaxMatrices];
    for (int i = 0; i < b.n; ++i) cycles[i] = plan(b.m[i], 1);
    for (int left = pairs - b.n; left > 0; --left) {
        int most = -1;
        for (int i = 0; i < b.n; ++i)
            if (b.m[i].pairs < most_units(b.m[i]) && (most < 0 || cycles[i] > cycles[most])) most = i;
        if (most < 0) break;
        cycles[most] = plan(b.m[most], b.m[most].pairs + 1);
    }
}

void describe(const gmc_matrix& g, Matrix& m);

// Describes the matrices of a launch and lays out its workspace; returns the workspace's size.
size_t lay_out(const gmc_matrix* matrices, const int* which, int n, uint8_t* workspace, Batch& b) {
    b.n = n;
    long long x_blocks = 0, gram_blocks = 0;
    b.norm_ctas = b.blocks = 0;
    bool splittable = false;
    for (int i = 0; i < n; ++i) {
        const gmc_matrix& g = matrices[which[i]];
        Matrix& m = b.m[i];
        describe(g, m);
        m.row_tiles = ceil_div(std::min(m.rows, m.cols), 128);
        m.col_blocks = 2 * ceil_div(std::max(m.rows, m.cols), 128);
        m.norm_first = b.norm_ctas;
        m.block_first = b.blocks;
        m.x_block = x_blocks;
        m.gram_block = gram_blocks;
        const long long blocks = (long long)m.row_tiles * m.col_blocks;
        b.norm_ctas += ceil_div(g.rows * g.cols, kNormElements);
        b.blocks += int(blocks);
        x_blocks += blocks;
        gram_blocks += 2LL * m.row_tiles * m.row_tiles;
        splittable = splittable || m.row_tiles <= 16;
    }
    size_t at = 0;
    auto take = [&](size_t size) {
        const size_t here = at;
        at += (size + 1023) & ~size_t(1023);
        return workspace + here;
    };
    b.x[0] = reinterpret_cast<__half*>(take(size_t(x_blocks) * kBlockBytes));
    b.x[1] = reinterpret_cast<__half*>(take(size_t(x_blocks) * kBlockBytes));
    b.gram = reinterpret_cast<__half*>(take(size_t(gram_blocks) * kBlockBytes));
    b.poly = reinterpret_cast<__half*>(take(size_t(gram_blocks) * kBlockBytes));
    b.squares = reinterpret_cast<double*>(take(size_t(b.norm_ctas) * sizeof(double)));
    // a matrix has no more tiles times shares than pairs, and none of 17 row tiles or more (9 x 10 / 2 tiles) has shares: the
    // size holds for any number of pairs up to kPairs
    b.partial = reinterpret_cast<float*>(take(splittable ? size_t(kPairs) * 256 * 256 * sizeof(float) : 0));
    b.arrived = reinterpret_cast<unsigned*>(take(size_t(n + 1) * sizeof(unsigned)));
    return at;
}

// The launch's plan: chunks, tiles, shares and pairs.
void make_plan(Batch& b, int pairs, bool fp32) {
    for (int i = 0; i < b.n; ++i) {
        const int rows = std::min(b.m[i].rows, b.m[i].cols);
        // fp32 results: against the plain fp32 evaluation's error, 256 x 4000 has 1.2 times with two stages and 2.3 with four,
        // 700 x 2000 0.9 with four and 1.6 with eight, 2048 x 2048 0.7 with eight and the time is 810, 720 and 680 us
        b.m[i].chunk = !fp32 ? kWholeAxis : rows <= 512 ? 2 : rows <= 1024 ? 4 : 8;
    }
    hand_out(b, pairs);
    // 16-bit results: one accumulation per sum while none is longer than 2048. The error before the last rounding is then 4e-6 to 2e-5
    // of the result (0.9 to 4 times the plain fp32 evaluation's; half a step is 2e-3 or 2.4e-4) and grows with the length
    // beyond: 4.8e-5 at 4095 x 6001, 8.7e-5 at 16384 x 32768 (random signs). In chunks of 1024 it is 1.4e-5 and 5e-6, and the
    // time 5.55 ms for 5.17 and 455 ms for 443; chunks of 2048 would take 5.42 ms for 2.7e-5, of 512 5.75 ms for 7e-6.
    b.whole = !fp32;
    for (int i = 0; i < b.n; ++i) b.whole = b.whole && longest_sum(b.m[i]) <= kWholeStages;
    if (!fp32 && !b.whole) {
        for (int i = 0; i < b.n; ++i) b.m[i].chunk = kLongChunk;
        hand_out(b, pairs);
    }
    b.pairs = 0;
    long long partials = 0;
    for (int i = 0; i < b.n; ++i) {
        Matrix& m = b.m[i];
        m.pair_first = b.pairs;
        b.pairs += m.pairs;
        m.partial_first = partials;
        if (m.splits > 1) partials += (long long)symmetric_tiles(m.row_tiles, m.gram_wide) * m.splits * 256 * (m.gram_wide ? 256 : 128);
    }
}

// Pairs of CTAs of the chain that the current device holds at once: a property of the device, asked for once per device.
int chain_pairs(int* pairs) {
    static std::atomic<int> known[64];
    int device = 0;
    GMC_CUDA_TRY(cudaGetDevice(&device));
    if (device < 64 && known[device].load() > 0) {
        *pairs = known[device].load();
        return GMC_OK;
    }
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(2 * kPairs);
    config.blockDim = dim3(kChainThreads);
    config.dynamicSmemBytes = kChainSmem;
    cudaLaunchAttribute attribute;
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = 2;
    attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    GMC_CUDA_TRY(cudaFuncSetAttribute(chain_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kChainSmem));
    GMC_CUDA_TRY(cudaOccupancyMaxActiveClusters(pairs, chain_kernel<false>, &config));       // one CTA per multiprocessor either way
    if (*pairs > kPairs) *pairs = kPairs;
    if (*pairs < kMaxMatrices) return GMC_ERR_UNSUPPORTED;
    if (device < 64) known[device].store(*pairs);
    return GMC_OK;
}

// The waits of the chain are bounded by 2^22 polls, 90 ms or more: a product of the largest matrix takes about 45 ms.
constexpr long long kMaxSide = 32768, kMaxShortSide = 16384;

int check_matrices(const gmc_matrix* matrices, int n) {
    if (n < 0 || (n > 0 && !matrices)) return n < 0 ? GMC_ERR_BAD_DIMS : GMC_ERR_NULL_POINTER;
    for (int i = 0; i < n; ++i) {
        const gmc_matrix& g = matrices[i];
        if (g.rows < 1 || g.cols < 1 || g.rows > kMaxSide || g.cols > kMaxSide || std::min(g.rows, g.cols) > kMaxShortSide) return GMC_ERR_BAD_DIMS;
        if (g.update_stride < g.cols || g.out_stride < g.cols) return GMC_ERR_BAD_DIMS;
    }
    return GMC_OK;
}

// Bounds of the iterates and of b A + c A A for singular values in [0, 1], and from them the planes' scales: powers of two
// that keep every value below the largest fp16 number. The extrema of x (a + b x^2 + c x^4) and of b l + c l^2, l = x^2, lie at
// the end of the interval or where the derivative is zero: at the roots of 5c l^2 + 3b l + a, of which one is taken from the
// product of both, so that nothing cancels however small c is (c = 0: the first is infinite), and at -b / 2c.
int make_polynomial(int steps, float a, float b, float c, Polynomial* out) {
    if (steps < 1 || steps > 32) return GMC_ERR_UNSUPPORTED;
    const double da = a, db = b, dc = c;
    if (!(fabs(da) < 100. && fabs(db) < 100. && fabs(dc) < 100.)) return GMC_ERR_UNSUPPORTED;
    const double q = -0.5 * (3. * db + copysign(sqrt(fmax(0., 9. * db * db - 20. * da * dc)), db));
    double top = 1., most = 1., poly = 0.;
    for (int s = 0; s < steps; ++s) {
        const double end = top * top;
        const double at[4] = {end, q / (5. * dc), da / q, -db / (2. * dc)};
        double next = 0.;
        for (double l : at) {
            if (!(l > 0. && l <= end)) continue;                      // infinite or not a number among others
            const double f = l * (db + dc * l);
            next = fmax(next, fabs(sqrt(l) * (da + f)));
            poly = fmax(poly, fabs(f));
        }
        if (!(next < 1.8)) return GMC_ERR_UNSUPPORTED;
        top = next;
        most = fmax(most, top);
    }
    auto scale_for = [](double most) { return exp2(floor(log2(60000. / most))); };
    const double sx = kScaleX, sa = scale_for(most * most), sp = scale_for(poly > 1e-3 ? poly : 1e-3);
    out->linear = dc == 0.;
    out->gram_factor = float(dc != 0. ? sa / (sx * sx) : db * sp / (sx * sx));
    out->poly_factor = float(dc * sp / (sa * sa));
    out->poly_from = float(db * sp / sa);
    out->step_factor = float(1. / sp);
    out->step_from = a;
    return GMC_OK;
}

template <typename T, bool MUON>
int run_batch(const Batch& b, int steps, const Polynomial& poly, float epsilon, const Momentum& mo, cudaStream_t stream) {
    norm_kernel<T, MUON><<<b.norm_ctas, 256, 0, stream>>>(b, mo);
    GMC_LAUNCH_CHECK();
    split_kernel<T, MUON><<<b.blocks, 256, 0, stream>>>(b, mo, epsilon);
    GMC_LAUNCH_CHECK();
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(unsigned(2 * b.pairs));
    config.blockDim = dim3(kChainThreads);
    config.dynamicSmemBytes = kChainSmem;
    config.stream = stream;
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeClusterDimension;
    attributes[0].val.clusterDim.x = 2;
    attributes[0].val.clusterDim.y = attributes[0].val.clusterDim.z = 1;
    attributes[1].id = cudaLaunchAttributeCooperative;
    attributes[1].val.cooperative = 1;
    config.attrs = attributes;
    config.numAttrs = 2;
    auto chain = b.whole ? chain_kernel<true> : chain_kernel<false>;
    GMC_CUDA_TRY(cudaFuncSetAttribute(chain, cudaFuncAttributeMaxDynamicSharedMemorySize, kChainSmem));
    GMC_CUDA_TRY(cudaLaunchKernelEx(&config, chain, b, steps, poly));
    finish_kernel<T, MUON><<<b.blocks, 256, 0, stream>>>(b, mo, steps & 1);
    GMC_LAUNCH_CHECK();
    return GMC_OK;
}

// Which kernel a matrix goes to, by its shape; the shared memory that it takes with a number of CTAs.
constexpr int kClusterSmemLimit = 227 * 1024 - 512;
int cluster_smem(int rows, int cols, int ranks) {
    return rows <= kShortRows ? int(short_smem(rows, cols, ranks)) + 1024 : mid_smem(mid_rows(rows), mid_blocks(cols, ranks));
}
bool fits(int rows, int cols, int ranks) {
    return cluster_smem(rows, cols, ranks) <= kClusterSmemLimit && (rows <= kShortRows || mid_blocks(cols, ranks) <= mid_max_blocks(mid_rows(rows)));
}
enum Kind { CLUSTER, CHAIN, KINDS };
Kind kind_of(const gmc_matrix& g) {
    const int rows = int(g.rows < g.cols ? g.rows : g.cols), cols = int(g.rows < g.cols ? g.cols : g.rows);
    return rows <= 128 && fits(rows, cols, 8) ? CLUSTER : CHAIN;
}
void describe(const gmc_matrix& g, Matrix& m) {
    m.update = g.update;
    m.momentum = g.momentum;
    m.out = g.out;
    m.update_stride = g.update_stride;
    m.out_stride = g.out_stride;
    m.rows = int(g.rows);
    m.cols = int(g.cols);
    m.rate = g.rate;
}

// One launch of clusters of `ranks` CTAs, one per matrix.
template <typename T, bool MUON>
int run_clusters(const gmc_matrix* matrices, const int* which, int n, int steps, float ca, float cb, float cc, const Polynomial& poly, float epsilon,
                 const Momentum& mo, cudaStream_t stream) {
    ClusterBatch b;
    int ranks = 1, smem = 0, device = 0, n_sm = 0;
    bool any_short = false;
    GMC_CUDA_TRY(cudaGetDevice(&device));
    GMC_CUDA_TRY(cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, device));
    for (int i = 0; i < n; ++i) {
        describe(matrices[which[i]], b.m[i]);
        const int rows = std::min(b.m[i].rows, b.m[i].cols), cols = std::max(b.m[i].rows, b.m[i].cols);
        any_short = any_short || rows <= kShortRows;
        // more CTAs where X does not fit, and while there are free multiprocessors beyond 256 columns a CTA: below, the exchange
        // of the shares costs more than the products save (64 x 160: 41 us with one CTA, 49 with four)
        while (ranks < 8 && (!fits(rows, cols, ranks) || (cols > 256 * ranks && 2 * ranks * n <= n_sm))) ranks *= 2;
    }
    // A CTA holds its multiprocessor's tensor memory: two clusters that shared two multiprocessors in different orders would wait
    // for each other's. A CTA of a cluster therefore takes more than half of the shared memory.
    if (ranks > 1) smem = 116 * 1024;
    for (int i = 0; i < n; ++i)
        smem = std::max(smem, cluster_smem(std::min(b.m[i].rows, b.m[i].cols), std::max(b.m[i].rows, b.m[i].cols), ranks));
    auto kernel = any_short ? cluster_kernel<T, MUON, true> : cluster_kernel<T, MUON, false>;
    GMC_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kClusterSmemLimit));
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(unsigned(n * ranks));
    config.blockDim = dim3(kMidThreads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attribute;
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = unsigned(ranks);
    attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    GMC_CUDA_TRY(cudaLaunchKernelEx(&config, kernel, b, ranks, mo, steps, ca, cb, cc, poly, epsilon));
    return GMC_OK;
}

template <typename T, bool MUON>
int run_typed(const gmc_matrix* matrices, int n, int steps, float ca, float cb, float cc, const Polynomial& poly, float epsilon, const Momentum& mo,
              void* workspace, size_t workspace_bytes, int pairs, cudaStream_t stream, int lost_wait) {
    int which[kMaxMatrices], count = 0;
    for (int kind = 0; kind < KINDS; ++kind) {
        for (int i = 0; i <= n; ++i) {
            if (i < n && kind_of(matrices[i]) == kind) which[count++] = i;
            if (count == kMaxMatrices || (i == n && count > 0)) {
                if (kind == CLUSTER) {
                    if (int s = run_clusters<T, MUON>(matrices, which, count, steps, ca, cb, cc, poly, epsilon, mo, stream)) return s;
                } else {
                    Batch b;
                    if (lay_out(matrices, which, count, static_cast<uint8_t*>(workspace), b) > workspace_bytes) return GMC_ERR_WORKSPACE;
                    make_plan(b, pairs, std::is_same<T, float>::value);
                    b.lost_wait = lost_wait;
                    if (int s = run_batch<T, MUON>(b, steps, poly, epsilon, mo, stream)) return s;
                }
                count = 0;
            }
        }
    }
    return GMC_OK;
}

size_t workspace_bytes_of(const gmc_matrix* matrices, int n) {
    int which[kMaxMatrices], count = 0;
    size_t most = 0;
    for (int i = 0; i <= n; ++i) {
        if (i < n && kind_of(matrices[i]) == CHAIN) which[count++] = i;
        if (count == kMaxMatrices || (i == n && count > 0)) {
            Batch b;
            most = std::max(most, lay_out(matrices, which, count, nullptr, b));
            count = 0;
        }
    }
    return most;
}

template <bool MUON>
int run(const gmc_matrix* matrices, int n, int dtype, int steps, float ca, float cb, float cc, float epsilon, const Momentum& mo,
        void* workspace, size_t workspace_bytes, void* stream, int lost_wait = -1) {
    if (int s = check_matrices(matrices, n)) return s;
    if (dtype < GMC_FLOAT32 || dtype > GMC_FLOAT16) return GMC_ERR_UNSUPPORTED;
    if (!(epsilon >= 1e-30f && epsilon <= 1e30f)) return GMC_ERR_UNSUPPORTED;
    Polynomial poly;
    if (int s = make_polynomial(steps, ca, cb, cc, &poly)) return s;
    for (int i = 0; i < n; ++i)
        if (!matrices[i].update || !matrices[i].out || (MUON && !matrices[i].momentum)) return GMC_ERR_NULL_POINTER;
    if (reinterpret_cast<uintptr_t>(workspace) & 1023u) return GMC_ERR_UNSUPPORTED;
    const size_t need = workspace_bytes_of(matrices, n);
    if (need > 0 && !workspace) return GMC_ERR_NULL_POINTER;
    if (need > workspace_bytes) return GMC_ERR_WORKSPACE;
    int pairs = 0;                                                    // asked for before anything is changed in place
    if (need > 0)
        if (int s = chain_pairs(&pairs)) return s;
    cudaStream_t cs = as_stream(stream);
    if (dtype == GMC_FLOAT32) return run_typed<float, MUON>(matrices, n, steps, ca, cb, cc, poly, epsilon, mo, workspace, workspace_bytes, pairs, cs, lost_wait);
    if (dtype == GMC_BFLOAT16) return run_typed<__nv_bfloat16, MUON>(matrices, n, steps, ca, cb, cc, poly, epsilon, mo, workspace, workspace_bytes, pairs, cs, lost_wait);
    return run_typed<__half, MUON>(matrices, n, steps, ca, cb, cc, poly, epsilon, mo, workspace, workspace_bytes, pairs, cs, lost_wait);
}

}  // namespace
}  // namespace gmc

GMC_DEFINE_TU_CHECK_WORD(newton_schulz)

extern "C" size_t gmc_orthogonalise_workspace_bytes(const gmc_matrix* matrices, int n_matrices) {
    using namespace gmc;
    if (check_matrices(matrices, n_matrices)) return 0;
    return workspace_bytes_of(matrices, n_matrices);
}

extern "C" int gmc_orthogonalise(const gmc_matrix* matrices, int n_matrices, int dtype, int steps, float a, float b, float c,
                                 float epsilon, void* workspace, size_t workspace_bytes, void* stream) {
    const gmc::Momentum none = {0.f, 1.f, 0, 1.f};
    return gmc::run<false>(matrices, n_matrices, dtype, steps, a, b, c, epsilon, none, workspace, workspace_bytes, stream);
}

extern "C" int gmc_debug_orthogonalise_lost_wait(const gmc_matrix* matrices, int n_matrices, int dtype, int steps, float a, float b, float c,
                                                 float epsilon, void* workspace, size_t workspace_bytes, int lost_wait, void* stream) {
    const gmc::Momentum none = {0.f, 1.f, 0, 1.f};
    return gmc::run<false>(matrices, n_matrices, dtype, steps, a, b, c, epsilon, none, workspace, workspace_bytes, stream, lost_wait);
}

extern "C" int gmc_muon_update(const gmc_matrix* matrices, int n_matrices, int dtype, int steps, float a, float b, float c,
                               float epsilon, double momentum, int nesterov, float decay, void* workspace, size_t workspace_bytes,
                               void* stream) {
    if (!(momentum >= 0. && momentum < 1.)) return GMC_ERR_UNSUPPORTED;
    // the new gradient's weight is rounded once: 1 - float(0.9999) would be off by 2e-4 of itself
    const gmc::Momentum mo = {float(momentum), float(1. - momentum), nesterov != 0, decay};
    return gmc::run<true>(matrices, n_matrices, dtype, steps, a, b, c, epsilon, mo, workspace, workspace_bytes, stream);
}
