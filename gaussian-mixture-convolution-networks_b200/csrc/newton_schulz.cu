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
// Layout. Planes lie in global memory as blocks of 128 rows x 64 columns in the exact byte order the tensor core reads from
// shared memory (128-byte swizzle), padded with zeros: loading an operand tile is one contiguous bulk copy, whatever the
// matrix's shape, and X serves both as rows (X X^T, K = columns) and across (B X, K = rows) without a transposed copy.
// A and A A are symmetric: only tiles on and below the diagonal are computed, their mirror images are stored with them.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tcgen05.cuh"

namespace gmc {
namespace {

namespace cg = cooperative_groups;

constexpr int kMaxMatrices = 48;                 // descriptors of one launch (kernel parameter)
constexpr int kBlockBytes = 128 * 64 * 2;        // one block of one plane
constexpr int kStageBytes = 4 * kBlockBytes;     // hi and lo of both operands, 64 wide in K
constexpr int kStages = 3;
constexpr int kProductSmem = kStages * kStageBytes + 1024;
constexpr float kScaleX = 32768.f, kScaleA = 32768.f, kScaleB = 16384.f;
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
    int norm_first, gram_first, step_first, block_first;      // first CTA of the matrix in each launch
    long long x_block, gram_block;                             // first block in the workspace's arrays
};
struct Batch {
    Matrix m[kMaxMatrices];
    int n;
    __half *x[2], *gram, *poly;
    double* partial;            // one per CTA of the norm
    int norm_ctas, gram_ctas, step_ctas, blocks;
};
struct Momentum {
    float beta, one_minus_beta;
    int nesterov;
    float decay;                // factor of the parameters
};

// The update's element: the given one, or the momentum's.
template <typename T>
__device__ __forceinline__ float load_float(const void* p, long long i) { return float(static_cast<const T*>(p)[i]); }

template <int Matrix::*FIRST>
__device__ __forceinline__ int find_matrix(const Batch& b, int cta) {
    int i = 0;
    while (i + 1 < b.n && cta >= b.m[i + 1].*FIRST) ++i;
    return i;
}

// Sum of squares of kNormElements elements per CTA, in fp64 (the squares of small updates leave the fp32 range); with a
// momentum the running average is updated on the way.
template <typename T, bool MUON>
__global__ void __launch_bounds__(256) norm_kernel(const __grid_constant__ Batch b, Momentum mo) {
    const int which = find_matrix<&Matrix::norm_first>(b, blockIdx.x);
    const Matrix& m = b.m[which];
    const long long total = (long long)m.rows * m.cols;
    const long long first = (long long)(int(blockIdx.x) - m.norm_first) * kNormElements;
    const int count = int(min((long long)kNormElements, total - first));
    const int row0 = int(first / m.cols), col0 = int(first - (long long)row0 * m.cols);
    double s = 0.;
    const unsigned cols = unsigned(m.cols);
#pragma unroll 4
    for (int i = threadIdx.x; i < count; i += 256) {
        const unsigned at = unsigned(col0 + i), r = at / cols;
        float u = load_float<T>(m.update, (row0 + (long long)r) * m.update_stride + (at - r * cols));
        if constexpr (MUON) {
            float* p = m.momentum + first + i;
            const float now = mo.beta * *p + mo.one_minus_beta * u;
            *p = now;
            u = mo.nesterov ? mo.one_minus_beta * u + mo.beta * now : now;
        }
        s += double(u) * double(u);
    }
    __shared__ double warp_sum[8];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0) warp_sum[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; ++w) s += warp_sum[w];
        b.partial[blockIdx.x] = s;
    }
}

__device__ __forceinline__ void split(float v, __half& hi, __half& lo) {
    hi = __float2half_rn(v);
    lo = __float2half_rn(v - __half2float(hi));
}
union Chunk {
    uint4 raw;
    __half h[8];
};

// X = U / (|U| + eps) as planes: one 128 x 64 block per CTA, padding included.
template <typename T, bool MUON>
__global__ void __launch_bounds__(256) split_kernel(const __grid_constant__ Batch b, Momentum mo, float epsilon) {
    const int which = find_matrix<&Matrix::block_first>(b, blockIdx.x);
    const Matrix& m = b.m[which];
    const int block = int(blockIdx.x) - m.block_first;
    const int norm_end = which + 1 < b.n ? b.m[which + 1].norm_first : b.norm_ctas;
    __shared__ double warp_sum[8];
    double s = 0.;
    for (int i = m.norm_first + threadIdx.x; i < norm_end; i += 256) s += b.partial[i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0) warp_sum[threadIdx.x >> 5] = s;
    __syncthreads();
    s = 0.;
    for (int w = 0; w < 8; ++w) s += warp_sum[w];
    const float norm = float(sqrt(s) + double(epsilon));
    const bool tall = m.rows > m.cols;
    const int wide_rows = tall ? m.cols : m.rows, wide_cols = tall ? m.rows : m.cols;
    const int row_tile = block / m.col_blocks, col_block = block - row_tile * m.col_blocks;
    const long long planes = (long long)m.row_tiles * m.col_blocks;
    uint8_t* hi_block = reinterpret_cast<uint8_t*>(b.x[0]) + (m.x_block + block) * kBlockBytes;
    uint8_t* lo_block = hi_block + planes * kBlockBytes;
    for (int i = threadIdx.x; i < 128 * 8; i += 256) {
        const int row = tall ? i & 127 : i >> 3, chunk = tall ? i >> 7 : i & 7;      // neighbouring threads read along a row
        const int r = row_tile * 128 + row;
        Chunk hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int c = col_block * 64 + chunk * 8 + e;
            float u = 0.f;
            if (r < wide_rows && c < wide_cols) {
                const long long rr = tall ? c : r, cc = tall ? r : c;
                u = load_float<T>(m.update, rr * m.update_stride + cc);
                if constexpr (MUON) {
                    const float now = m.momentum[rr * m.cols + cc];
                    u = mo.nesterov ? mo.one_minus_beta * u + mo.beta * now : now;
                }
                u = u / norm * kScaleX;
            }
            split(u, hi.h[e], lo.h[e]);
        }
        const uint32_t at = swizzled_offset(row, chunk);
        *reinterpret_cast<uint4*>(hi_block + at) = hi.raw;
        *reinterpret_cast<uint4*>(lo_block + at) = lo.raw;
    }
}

// The last X as the output's type, or subtracted from the parameters.
template <typename T, bool MUON>
__global__ void __launch_bounds__(256) finish_kernel(const __grid_constant__ Batch b, Momentum mo, int which_x) {
    const int which = find_matrix<&Matrix::block_first>(b, blockIdx.x);
    const Matrix& m = b.m[which];
    const int block = int(blockIdx.x) - m.block_first;
    const bool tall = m.rows > m.cols;
    const int wide_rows = tall ? m.cols : m.rows, wide_cols = tall ? m.rows : m.cols;
    const int row_tile = block / m.col_blocks, col_block = block - row_tile * m.col_blocks;
    const long long planes = (long long)m.row_tiles * m.col_blocks;
    const uint8_t* hi_block = reinterpret_cast<const uint8_t*>(b.x[which_x]) + (m.x_block + block) * kBlockBytes;
    const uint8_t* lo_block = hi_block + planes * kBlockBytes;
    T* out = static_cast<T*>(m.out);
    for (int i = threadIdx.x; i < 128 * 8; i += 256) {
        const int row = tall ? i & 127 : i >> 3, chunk = tall ? i >> 7 : i & 7;
        const int r = row_tile * 128 + row;
        if (r >= wide_rows) continue;
        const uint32_t at = swizzled_offset(row, chunk);
        Chunk hi, lo;
        hi.raw = *reinterpret_cast<const uint4*>(hi_block + at);
        lo.raw = *reinterpret_cast<const uint4*>(lo_block + at);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int c = col_block * 64 + chunk * 8 + e;
            if (c >= wide_cols) break;
            const long long o = tall ? c * m.out_stride + r : r * m.out_stride + c;
            const float x = (__half2float(hi.h[e]) + __half2float(lo.h[e])) * (1.f / kScaleX);
            out[o] = T(MUON ? float(out[o]) * mo.decay - m.rate * x : x);
        }
    }
}

enum Product { GRAM, POLY, STEP };

// One 128 x kTileN tile of a product per CTA. Warps 0-7 write the tile (warp w: rows 32 (w % 4) .. + 31, half w / 4 of the
// columns), warp 8 loads (bulk copies into a ring of stages), warp 9 issues the MMAs.
//
// The tensor core adds into its fp32 accumulator without rounding to nearest, which over a long inner axis drifts (7e-6 of
// the result at 2000 columns). hi hi is therefore accumulated over kChunk stages only and then added to registers, while
// the MMAs of the next chunk's mixed products run; hi lo and lo hi, 2^-11 as large, have an accumulator of their own.
constexpr int kTileN = 128;
constexpr int kWriters = 256;
constexpr int kProductThreads = kWriters + 64;
constexpr int kChunk = 2;                         // stages, 64 wide in K each
template <Product P>
__global__ void __launch_bounds__(kProductThreads, 1) product_kernel(const __grid_constant__ Batch b, int from_x, float c0, float c1) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[kStages], empty[kStages], ready, drained, done;
    __shared__ uint32_t tmem_address;
    __shared__ int failed;
    const uint32_t pad = (1024u - (smem_u32(smem_raw) & 1023u)) & 1023u;
    uint8_t* stages = smem_raw + pad;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    constexpr bool symmetric = P != STEP;
    const int which = find_matrix<symmetric ? &Matrix::gram_first : &Matrix::step_first>(b, blockIdx.x);
    const Matrix& m = b.m[which];
    int tile = int(blockIdx.x) - (symmetric ? m.gram_first : m.step_first);
    int ti, tj;                                                       // tile row, tile column
    if (symmetric) {
        ti = int((sqrtf(8.f * float(tile) + 1.f) - 1.f) * 0.5f);
        while (ti * (ti + 1) / 2 > tile) --ti;
        while ((ti + 1) * (ti + 2) / 2 <= tile) ++ti;
        tj = tile - ti * (ti + 1) / 2;
    } else {
        const int col_tiles = m.col_blocks >> 1;
        ti = tile / col_tiles;
        tj = tile - ti * col_tiles;
    }
    const int gram_blocks = 2 * m.row_tiles;                          // column blocks of A and B
    const long long x_plane = (long long)m.row_tiles * m.col_blocks * kBlockBytes;
    const long long gram_plane = (long long)m.row_tiles * gram_blocks * kBlockBytes;
    const uint8_t* x = reinterpret_cast<const uint8_t*>(b.x[from_x]) + m.x_block * kBlockBytes;
    uint8_t* x_out = reinterpret_cast<uint8_t*>(b.x[from_x ^ 1]) + m.x_block * kBlockBytes;
    uint8_t* gram = reinterpret_cast<uint8_t*>(b.gram) + m.gram_block * kBlockBytes;
    uint8_t* poly = reinterpret_cast<uint8_t*>(b.poly) + m.gram_block * kBlockBytes;
    const int k_blocks = P == GRAM ? m.col_blocks : gram_blocks;      // even
    const int chunks = k_blocks / kChunk;

    if (tid == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(&ready, 1);
        mbar_init(&drained, kWriters / 32);
        mbar_init(&done, 1);
        failed = 0;
        fence_mbar_init();
    }
    if (warp == kWriters / 32 + 1) tmem_alloc(&tmem_address, 2 * kTileN);
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t main_sum = tmem_address, mixed_sum = tmem_address + kTileN;

    if (tid == kWriters) {
        bool ok = true;
        int issued = 0;
        for (int kb = 0; kb < k_blocks; ++kb) {
            const int s = kb % kStages;
            if (kb >= kStages && !(ok = mbar_wait_bounded(&empty[s], ((kb / kStages) - 1) & 1))) break;
            uint8_t* stage = stages + s * kStageBytes;
            mbar_arrive_expect_tx(&full[s], kStageBytes);
            const uint8_t* a;
            long long plane;
            if (P == GRAM) a = x + ((long long)ti * m.col_blocks + kb) * kBlockBytes, plane = x_plane;
            else a = (P == POLY ? gram : poly) + ((long long)ti * gram_blocks + kb) * kBlockBytes, plane = gram_plane;
            bulk_copy_g2s(stage, a, kBlockBytes, &full[s]);
            bulk_copy_g2s(stage + kBlockBytes, a + plane, kBlockBytes, &full[s]);
            if (P == STEP) {
                // 64 rows of two neighbouring column blocks of X, each half a block
                const uint8_t* xb = x + ((long long)(kb >> 1) * m.col_blocks + 2 * tj) * kBlockBytes + (kb & 1) * (kBlockBytes / 2);
                for (int q = 0; q < 4; ++q)
                    bulk_copy_g2s(stage + 2 * kBlockBytes + q * (kBlockBytes / 2), xb + (q >> 1) * x_plane + (long long)(q & 1) * kBlockBytes,
                                  kBlockBytes / 2, &full[s]);
            } else {
                const uint8_t* r = P == GRAM ? x + ((long long)tj * m.col_blocks + kb) * kBlockBytes
                                             : gram + ((long long)tj * gram_blocks + kb) * kBlockBytes;
                bulk_copy_g2s(stage + 2 * kBlockBytes, r, kBlockBytes, &full[s]);
                bulk_copy_g2s(stage + 3 * kBlockBytes, r + plane, kBlockBytes, &full[s]);
            }
            issued = kb + 1;
        }
        if (!ok) {
            *(volatile int*)&failed = 1;
            for (int kb = max(0, issued - kStages); kb < issued; ++kb) mbar_wait_bounded(&full[kb % kStages], (kb / kStages) & 1);
        }
    } else if (tid == kWriters + 32) {
        constexpr uint32_t instruction = f16_instruction(128, kTileN, P == STEP);
        bool ok = true;
        for (int kb = 0; kb < k_blocks; ++kb) {
            const int s = kb % kStages, chunk = kb / kChunk;
            if (!(ok = mbar_wait_bounded(&full[s], (kb / kStages) & 1))) break;
            tmem_fence_after();
            const uint32_t stage = smem_u32(stages + s * kStageBytes);
            auto a_of = [&](int plane, int k) { return k_major_descriptor(stage + plane * kBlockBytes + k * 32); };
            auto b_of = [&](int plane, int k) {
                return P == STEP ? mn_major_descriptor(stage + (2 + plane) * kBlockBytes + k * 2048, kBlockBytes / 2)
                                 : k_major_descriptor(stage + (2 + plane) * kBlockBytes + k * 32);
            };
#pragma unroll
            for (int k = 0; k < 4; ++k) {                             // 16 of the 64 in K
                mma_f16(mixed_sum, a_of(0, k), b_of(1, k), instruction, kb > 0 || k > 0);
                mma_f16(mixed_sum, a_of(1, k), b_of(0, k), instruction, true);
            }
            if (kb % kChunk == 0 && chunk > 0) {
                if (!(ok = mbar_wait_bounded(&drained, (chunk - 1) & 1))) break;
                tmem_fence_after();
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) mma_f16(main_sum, a_of(0, k), b_of(0, k), instruction, kb % kChunk > 0 || k > 0);
            mma_commit(&empty[s]);
            if (kb % kChunk == kChunk - 1) mma_commit(&ready);
        }
        if (!ok) *(volatile int*)&failed = 1;
        mma_commit(&done);
        mbar_wait_bounded(&done, 0);                                  // nothing of this CTA in flight when its TMEM is freed
    } else if (warp < kWriters / 32) {
        constexpr int C = kTileN / 2;                                 // columns of a warp
        const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
        const int col0 = (warp >> 2) * C;
        float sum[C];
#pragma unroll
        for (int i = 0; i < C; ++i) sum[i] = 0.f;
        bool complete = true;
        for (int chunk = 0; chunk < chunks && complete; ++chunk) {
            complete = mbar_wait_bounded(&ready, chunk & 1);
            tmem_fence_after();
#pragma unroll
            for (int q = 0; q < C; q += 32) {
                float v[32];
                tmem_load32(main_sum + lanes + col0 + q, v);
#pragma unroll
                for (int i = 0; i < 32; ++i) sum[q + i] += v[i];
            }
            tmem_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&drained);
        }
        complete = complete && *(volatile int*)&failed == 0;
        const int row = (warp & 3) * 32 + lane;
        const long long plane = P == STEP ? x_plane : gram_plane;
#pragma unroll
        for (int q = 0; q < C; q += 32) {                             // 32 columns at a time
            float v[32];
            tmem_load32(mixed_sum + lanes + col0 + q, v);
            const int col = col0 + q;
            const long long to_block = (P == STEP ? (long long)ti * m.col_blocks + (kTileN / 64) * tj
                                                  : (long long)ti * gram_blocks + (kTileN / 64) * tj) + (col >> 6);
            uint8_t* to = (P == GRAM ? gram : P == POLY ? poly : x_out) + to_block * kBlockBytes;
            const uint8_t* from = (P == POLY ? gram : x) + to_block * kBlockBytes;
#pragma unroll
            for (int g = 0; g < 4; ++g) {                             // 8 columns = one 16-byte chunk
                const uint32_t at = swizzled_offset(row, ((col & 63) >> 3) + g);
                Chunk hi, lo, from_hi, from_lo;
                if (P != GRAM) {
                    from_hi.raw = *reinterpret_cast<const uint4*>(from + at);
                    from_lo.raw = *reinterpret_cast<const uint4*>(from + plane + at);
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float r = (sum[q + g * 8 + e] + v[g * 8 + e]) * c1;
                    if (P != GRAM) r += c0 * (__half2float(from_hi.h[e]) + __half2float(from_lo.h[e]));
                    if (!complete) r = __int_as_float(0x7fffffff);
                    split(r, hi.h[e], lo.h[e]);
                }
                *reinterpret_cast<uint4*>(to + at) = hi.raw;
                *reinterpret_cast<uint4*>(to + plane + at) = lo.raw;
                if (symmetric && ti != tj) {
                    uint8_t* mirror = (P == GRAM ? gram : poly) + ((long long)tj * gram_blocks + 2 * ti + (row >> 6)) * kBlockBytes;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint32_t to_at = swizzled_offset(col + g * 8 + e, (row & 63) >> 3) + (row & 7) * 2;
                        *reinterpret_cast<__half*>(mirror + to_at) = hi.h[e];
                        *reinterpret_cast<__half*>(mirror + plane + to_at) = lo.h[e];
                    }
                }
            }
        }
        tmem_fence_before();
    }
    __syncthreads();
    if (warp == kWriters / 32 + 1) {
        tmem_fence_after();
        tmem_free(tmem_address, 2 * kTileN);
    }
}

// ---- matrices with a short side: the whole chain in one launch, fp32 -------------------------------------------------
// One cluster per matrix. Each CTA keeps X for its share of the columns in shared memory over all steps; per step every CTA
// adds up all shares of X X^T over distributed shared memory, forms P = a I + b A + c A A for itself and multiplies its own
// columns with it in place. Nothing goes through global memory between
// the update's elements and the result, there is one launch instead of three per step, and the products are fp32.
constexpr int kShortThreads = 512;
constexpr int kShortWarps = kShortThreads / 32;
constexpr int kShortRows = 64;
struct ShortBatch {
    Matrix m[kMaxMatrices];
};
// Sizes for X padded to MP rows: 4 x 4 tiles on and below the diagonal of X X^T, and groups of threads that share its sums.
__host__ __device__ constexpr int short_padded_rows(int rows) { return rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }
__host__ __device__ constexpr int short_tiles(int mp) { return (mp / 4) * (mp / 4 + 1) / 2; }
__host__ __device__ constexpr int short_packed(int mp) { return short_tiles(mp) * 16; }
__host__ __device__ constexpr int short_groups(int mp) { return mp == 64 ? kShortThreads / short_tiles(64) : 1; }
__host__ __device__ constexpr int short_columns(int cols, int ranks) { return ((cols + ranks - 1) / ranks + 3) & ~3; }
__host__ __device__ constexpr int short_pitch(int columns) { return ((columns + 27) / 32) * 32 + 4; }    // = 4 mod 32 banks, >= columns
__host__ __device__ constexpr size_t short_smem(int rows, int cols, int ranks) {
    const int mp = short_padded_rows(rows);
    return size_t(mp * short_pitch(short_columns(cols, ranks)) + 2 * mp * (mp + 4) + (2 + short_groups(mp)) * short_packed(mp)) * sizeof(float);
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
// MP = 64: a thread per tile and group of columns, the groups' sums added through shared memory; smaller: a warp per tile,
// its lanes share the columns. done(e, value) is called once for every packed element.
template <int MP, typename Done>
__device__ __forceinline__ void symmetric_product(const float* from, int pitch, int length, float* partial, Done&& done) {
    constexpr int side = MP / 4, tiles = short_tiles(MP), packed = short_packed(MP), groups = short_groups(MP);
    const int tid = threadIdx.x;
    if constexpr (groups > 1) {
        const int tile = tid % tiles, group = tid / tiles;
        if (group < groups) {
            int ti, tj;
            tile_place(tile, ti, tj);
            float acc[16] = {};
            tile_product(acc, from + ti * pitch, from + tj * pitch, side * pitch, group * 4, groups * 4, length);
#pragma unroll
            for (int i = 0; i < 16; ++i) partial[group * packed + i * tiles + tile] = acc[i];
        }
        __syncthreads();
        constexpr int each = (packed + kShortThreads - 1) / kShortThreads;
        float v[each];
#pragma unroll
        for (int i = 0; i < each; ++i) {
            const int e = tid + i * kShortThreads;
            v[i] = 0.f;
#pragma unroll
            for (int g = 0; g < groups; ++g) v[i] += e < packed ? partial[g * packed + e] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < each; ++i)
            if (tid + i * kShortThreads < packed) done(tid + i * kShortThreads, v[i]);
    } else {
        const int lane = tid & 31;
        for (int tile = tid >> 5; tile < tiles; tile += kShortWarps) {
            int ti, tj;
            tile_place(tile, ti, tj);
            float acc[16] = {};
            tile_product(acc, from + ti * pitch, from + tj * pitch, side * pitch, lane * 4, 128, length);
            const float v = warp_sum16(acc, lane);
            if ((lane & 1) == 0) done((lane >> 1) * tiles + tile, v);
        }
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
    float* partial = share + 2 * packed;

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
            u[j] = in ? load_float<T>(m.update, (first_row + o) * m.update_stride + first + i) : 0.f;
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
    const float factor = float(1. / (sqrt(s) + double(epsilon)));
    for (int i = tid * 4; i < MP * pitch; i += kShortThreads * 4) {
        float4 v = *reinterpret_cast<float4*>(x + i);
        v.x *= factor, v.y *= factor, v.z *= factor, v.w *= factor;
        *reinterpret_cast<float4*>(x + i) = v;
    }
    // where this thread's elements of the packed sums go (the same in every step)
    constexpr int each = (packed + kShortThreads - 1) / kShortThreads;
    int at[each], mirror[each];
#pragma unroll
    for (int i = 0; i < each; ++i) packed_places<MP>(min(tid + i * kShortThreads, packed - 1), gp, at[i], mirror[i]);
    __syncthreads();

    for (int step = 0; step < steps; ++step) {
        // A: every CTA adds up all shares in their order. A share's buffer is written again two steps, so one barrier, later.
        float* mine = share + (step & 1) * packed;
        symmetric_product<MP>(x, pitch, columns, partial, [&](int e, float v) { mine[e] = v; });
        if (ranks > 1) cluster.sync();
        else __syncthreads();
        float v[each];
#pragma unroll
        for (int i = 0; i < each; ++i) v[i] = 0.f;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            if (q < ranks) {
                const float* theirs = ranks > 1 ? cluster.map_shared_rank(mine, q) : mine;
#pragma unroll
                for (int i = 0; i < each; ++i) v[i] += theirs[min(tid + i * kShortThreads, packed - 1)];
            }
        }
#pragma unroll
        for (int i = 0; i < each; ++i)
            if (tid + i * kShortThreads < packed) gram[at[i]] = gram[mirror[i]] = v[i];
        __syncthreads();
        symmetric_product<MP>(gram, gp, MP, partial, [&](int e, float v) {
            int a, b;
            if constexpr (short_groups(MP) > 1) {
                const int i = (e - tid) / kShortThreads;
                a = b = 0;
#pragma unroll
                for (int j = 0; j < each; ++j)
                    if (i == j) a = at[j], b = mirror[j];
            } else {
                packed_places<MP>(e, gp, a, b);
            }
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

template <typename T, bool MUON>
__global__ void __launch_bounds__(kShortThreads, 1) short_kernel(const __grid_constant__ ShortBatch b, int ranks, Momentum mo, int steps, float ca,
                                                                 float cb, float cc, float epsilon) {
    extern __shared__ __align__(16) float smem[];
    __shared__ double warp_sum[kShortWarps], cta_sum;
    const Matrix& m = b.m[blockIdx.x / unsigned(ranks)];
    const int rank = int(blockIdx.x % unsigned(ranks)), rows = min(m.rows, m.cols);
    if (rows <= 8) short_matrix<T, MUON, 8>(m, ranks, rank, mo, steps, ca, cb, cc, epsilon, smem, warp_sum, &cta_sum);
    else if (rows <= 16) short_matrix<T, MUON, 16>(m, ranks, rank, mo, steps, ca, cb, cc, epsilon, smem, warp_sum, &cta_sum);
    else if (rows <= 32) short_matrix<T, MUON, 32>(m, ranks, rank, mo, steps, ca, cb, cc, epsilon, smem, warp_sum, &cta_sum);
    else short_matrix<T, MUON, 64>(m, ranks, rank, mo, steps, ca, cb, cc, epsilon, smem, warp_sum, &cta_sum);
}

// ---- host side -------------------------------------------------------------------------------------------------------
int ceil_div(long long a, long long b) { return int((a + b - 1) / b); }

void fill(const gmc_matrix* matrices, const int* which, int n, Batch* batch, size_t* bytes, uint8_t* workspace) {
    Batch& b = *batch;
    b.n = n;
    long long x_blocks = 0, gram_blocks = 0;
    b.norm_ctas = b.gram_ctas = b.step_ctas = b.blocks = 0;
    for (int i = 0; i < n; ++i) {
        const gmc_matrix& g = matrices[which[i]];
        Matrix& m = b.m[i];
        const long long wide_rows = g.rows < g.cols ? g.rows : g.cols, wide_cols = g.rows < g.cols ? g.cols : g.rows;
        m.update = g.update;
        m.momentum = g.momentum;
        m.out = g.out;
        m.update_stride = g.update_stride;
        m.out_stride = g.out_stride;
        m.rows = int(g.rows);
        m.cols = int(g.cols);
        m.rate = g.rate;
        m.row_tiles = ceil_div(wide_rows, 128);
        m.col_blocks = 2 * ceil_div(wide_cols, 128);
        m.norm_first = b.norm_ctas;
        m.gram_first = b.gram_ctas;
        m.step_first = b.step_ctas;
        m.block_first = b.blocks;
        m.x_block = x_blocks;
        m.gram_block = gram_blocks;
        const long long blocks = (long long)m.row_tiles * m.col_blocks;
        b.norm_ctas += ceil_div(g.rows * g.cols, kNormElements);
        b.gram_ctas += m.row_tiles * (m.row_tiles + 1) / 2;
        b.step_ctas += int(blocks / 2);
        b.blocks += int(blocks);
        x_blocks += 2 * blocks;
        gram_blocks += 2LL * m.row_tiles * 2 * m.row_tiles;
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
    b.partial = reinterpret_cast<double*>(take(size_t(b.norm_ctas) * sizeof(double)));
    *bytes = at;
}

constexpr long long kMaxSide = 32768;

int check_matrices(const gmc_matrix* matrices, int n) {
    if (n < 0 || (n > 0 && !matrices)) return n < 0 ? GMC_ERR_BAD_DIMS : GMC_ERR_NULL_POINTER;
    for (int i = 0; i < n; ++i) {
        const gmc_matrix& g = matrices[i];
        if (g.rows < 1 || g.cols < 1 || g.rows > kMaxSide || g.cols > kMaxSide) return GMC_ERR_BAD_DIMS;
        if (g.update_stride < g.cols || g.out_stride < g.cols) return GMC_ERR_BAD_DIMS;
    }
    return GMC_OK;
}

// Bounds of the iterates on [0, 1]: the planes' scales leave room for |X| < 1.4 and |b A + c A A| < 3.9. The extrema of
// x (a + b x^2 + c x^4) and b l + c l^2 lie at the end of the interval or where the derivative is zero.
int check_polynomial(int steps, float a, float b, float c) {
    if (steps < 1 || steps > 32) return GMC_ERR_UNSUPPORTED;
    const double da = a, db = b, dc = c;
    const double root = sqrt(fmax(0., 9. * db * db - 20. * da * dc));
    double top = 1.;
    for (int s = 0; s < steps; ++s) {
        const double end = top * top;
        const double at[4] = {end, (-3. * db + root) / (10. * dc), (-3. * db - root) / (10. * dc), -db / (2. * dc)};
        double next = 0., poly = 0.;
        for (double l : at) {
            if (dc == 0. && l != end) l = db != 0. ? -da / (3. * db) : end;
            if (!(l > 0. && l <= end)) continue;
            next = fmax(next, fabs(sqrt(l) * (da + l * (db + dc * l))));
            poly = fmax(poly, fabs(l * (db + dc * l)));
        }
        if (!(poly < 3.9) || !(next < 1.4)) return GMC_ERR_UNSUPPORTED;
        top = next;
    }
    return da == da && db == db && dc == dc ? GMC_OK : GMC_ERR_UNSUPPORTED;
}

template <typename T, bool MUON>
int run_batch(const Batch& b, int steps, float ca, float cb, float cc, float epsilon, const Momentum& mo, cudaStream_t stream) {
    norm_kernel<T, MUON><<<b.norm_ctas, 256, 0, stream>>>(b, mo);
    GMC_LAUNCH_CHECK();
    split_kernel<T, MUON><<<b.blocks, 256, 0, stream>>>(b, mo, epsilon);
    GMC_LAUNCH_CHECK();
    GMC_CUDA_TRY(cudaFuncSetAttribute(product_kernel<GRAM>, cudaFuncAttributeMaxDynamicSharedMemorySize, kProductSmem));
    GMC_CUDA_TRY(cudaFuncSetAttribute(product_kernel<POLY>, cudaFuncAttributeMaxDynamicSharedMemorySize, kProductSmem));
    GMC_CUDA_TRY(cudaFuncSetAttribute(product_kernel<STEP>, cudaFuncAttributeMaxDynamicSharedMemorySize, kProductSmem));
    int x = 0;
    for (int s = 0; s < steps; ++s, x ^= 1) {
        product_kernel<GRAM><<<b.gram_ctas, kProductThreads, kProductSmem, stream>>>(b, x, 0.f, kScaleA / (kScaleX * kScaleX));
        GMC_LAUNCH_CHECK();
        product_kernel<POLY><<<b.gram_ctas, kProductThreads, kProductSmem, stream>>>(b, x, cb * (kScaleB / kScaleA), cc * (kScaleB / (kScaleA * kScaleA)));
        GMC_LAUNCH_CHECK();
        product_kernel<STEP><<<b.step_ctas, kProductThreads, kProductSmem, stream>>>(b, x, ca, 1.f / kScaleB);
        GMC_LAUNCH_CHECK();
    }
    finish_kernel<T, MUON><<<b.blocks, 256, 0, stream>>>(b, mo, x);
    GMC_LAUNCH_CHECK();
    return GMC_OK;
}

// A matrix goes to the one-launch kernel if its short side fits the tile grid and X fits the shared memory of eight CTAs.
constexpr size_t kShortSmemLimit = 220 * 1024;
bool is_short(const gmc_matrix& g) {
    const long long rows = g.rows < g.cols ? g.rows : g.cols, cols = g.rows < g.cols ? g.cols : g.rows;
    return rows <= kShortRows && short_smem(int(rows), int(cols), 8) <= kShortSmemLimit;
}

template <typename T, bool MUON>
int run_short(const gmc_matrix* matrices, const int* which, int n, int steps, float ca, float cb, float cc, float epsilon,
              const Momentum& mo, cudaStream_t stream) {
    ShortBatch b;
    int ranks = 1, device = 0, n_sm = 0;
    GMC_CUDA_TRY(cudaGetDevice(&device));
    GMC_CUDA_TRY(cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, device));
    size_t smem = 0;
    for (int i = 0; i < n; ++i) {
        const gmc_matrix& g = matrices[which[i]];
        Matrix& m = b.m[i];
        m.update = g.update;
        m.momentum = g.momentum;
        m.out = g.out;
        m.update_stride = g.update_stride;
        m.out_stride = g.out_stride;
        m.rows = int(g.rows);
        m.cols = int(g.cols);
        m.rate = g.rate;
        const int rows = m.rows < m.cols ? m.rows : m.cols, cols = m.rows < m.cols ? m.cols : m.rows;
        while (ranks < 8 && ((cols / ranks > 40 && 2 * ranks * n <= n_sm) || short_smem(rows, cols, ranks) > kShortSmemLimit)) ranks *= 2;
    }
    for (int i = 0; i < n; ++i) {
        const int rows = b.m[i].rows < b.m[i].cols ? b.m[i].rows : b.m[i].cols, cols = b.m[i].rows < b.m[i].cols ? b.m[i].cols : b.m[i].rows;
        const size_t need = short_smem(rows, cols, ranks);
        smem = need > smem ? need : smem;
    }
    GMC_CUDA_TRY(cudaFuncSetAttribute(short_kernel<T, MUON>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kShortSmemLimit)));
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(unsigned(n * ranks));
    config.blockDim = dim3(kShortThreads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attribute;
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = unsigned(ranks);
    attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    GMC_CUDA_TRY(cudaLaunchKernelEx(&config, short_kernel<T, MUON>, b, ranks, mo, steps, ca, cb, cc, epsilon));
    return GMC_OK;
}

template <typename T, bool MUON>
int run_typed(const gmc_matrix* matrices, int n, int steps, float ca, float cb, float cc, float epsilon, const Momentum& mo,
              void* workspace, size_t workspace_bytes, cudaStream_t stream) {
    int which[kMaxMatrices], count = 0;
    for (int pass = 0; pass < 2; ++pass) {
        for (int i = 0; i <= n; ++i) {
            if (i < n && is_short(matrices[i]) == (pass == 0)) which[count++] = i;
            if (count == kMaxMatrices || (i == n && count > 0)) {
                if (pass == 0) {
                    if (int s = run_short<T, MUON>(matrices, which, count, steps, ca, cb, cc, epsilon, mo, stream)) return s;
                } else {
                    Batch b;
                    size_t bytes = 0;
                    fill(matrices, which, count, &b, &bytes, static_cast<uint8_t*>(workspace));
                    if (bytes > workspace_bytes) return GMC_ERR_WORKSPACE;
                    if (int s = run_batch<T, MUON>(b, steps, ca, cb, cc, epsilon, mo, stream)) return s;
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
        if (i < n && !is_short(matrices[i])) which[count++] = i;
        if (count == kMaxMatrices || (i == n && count > 0)) {
            Batch b;
            size_t bytes = 0;
            fill(matrices, which, count, &b, &bytes, nullptr);
            most = bytes > most ? bytes : most;
            count = 0;
        }
    }
    return most;
}

template <bool MUON>
int run(const gmc_matrix* matrices, int n, int dtype, int steps, float ca, float cb, float cc, float epsilon, const Momentum& mo,
        void* workspace, size_t workspace_bytes, void* stream) {
    if (int s = check_matrices(matrices, n)) return s;
    if (dtype < GMC_FLOAT32 || dtype > GMC_FLOAT16) return GMC_ERR_UNSUPPORTED;
    if (!(epsilon >= 1e-30f && epsilon <= 1e30f)) return GMC_ERR_UNSUPPORTED;
    if (int s = check_polynomial(steps, ca, cb, cc)) return s;
    for (int i = 0; i < n; ++i)
        if (!matrices[i].update || !matrices[i].out || (MUON && !matrices[i].momentum)) return GMC_ERR_NULL_POINTER;
    if (reinterpret_cast<uintptr_t>(workspace) & 1023u) return GMC_ERR_UNSUPPORTED;
    const size_t need = workspace_bytes_of(matrices, n);
    if (need > 0 && !workspace) return GMC_ERR_NULL_POINTER;
    if (need > workspace_bytes) return GMC_ERR_WORKSPACE;
    cudaStream_t cs = as_stream(stream);
    if (dtype == GMC_FLOAT32) return run_typed<float, MUON>(matrices, n, steps, ca, cb, cc, epsilon, mo, workspace, workspace_bytes, cs);
    if (dtype == GMC_BFLOAT16) return run_typed<__nv_bfloat16, MUON>(matrices, n, steps, ca, cb, cc, epsilon, mo, workspace, workspace_bytes, cs);
    return run_typed<__half, MUON>(matrices, n, steps, ca, cb, cc, epsilon, mo, workspace, workspace_bytes, cs);
}

}  // namespace
}  // namespace gmc

GMC_DEFINE_TU_CHECK_READER(newton_schulz)

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

extern "C" int gmc_muon_update(const gmc_matrix* matrices, int n_matrices, int dtype, int steps, float a, float b, float c,
                               float epsilon, float momentum, int nesterov, float decay, void* workspace, size_t workspace_bytes,
                               void* stream) {
    if (!(momentum >= 0.f && momentum < 1.f)) return GMC_ERR_UNSUPPORTED;
    const gmc::Momentum mo = {momentum, 1.f - momentum, nesterov != 0, decay};
    return gmc::run<true>(matrices, n_matrices, dtype, steps, a, b, c, epsilon, mo, workspace, workspace_bytes, stream);
}
