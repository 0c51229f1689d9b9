// Selection of key blocks for block-sparse attention: the means of blocks of
// rows, the products of the means, and the top-k of each (head, query block).
//
// A selection hangs on differences between scores, so nothing here may depend
// on the order of a sum: means are summed in 64 bits (bf16 values of one block
// add up exactly there) and rounded once to 32 bits; scores are sums of exact
// products in 64 bits; equal scores go to the lowest index.  A NaN score ranks
// below every number, -0 equals +0.
#include "common.cuh"

namespace h3b {
namespace sel {

constexpr int kThreads = 256;

// mean over the rows of a block of x [S, H, D] -> out [nb, H, D] fp32.
// One CTA per (block, head); 8 channels a thread, kThreads / (D / 8) row lanes.
template <int D>
__global__ void __launch_bounds__(kThreads) means_kernel(const uint16_t* __restrict__ x, int64_t ld, int64_t hs,
                                                         int64_t S, int H, int rows, float* __restrict__ out) {
    constexpr int kCols = D / 8;
    constexpr int kRows = kThreads / kCols;
    const int h = (int)(blockIdx.x % (unsigned)H);
    const int64_t b = blockIdx.x / (unsigned)H;
    const int col = threadIdx.x % kCols, row = threadIdx.x / kCols;
    const int count = (int)min((int64_t)rows, S - b * rows);
    const uint16_t* src = x + b * rows * ld + h * hs + col * 8;
    double acc[8] = {};
#pragma unroll 4
    for (int r = row; r < count; r += kRows) {
        const uint4 v = *reinterpret_cast<const uint4*>(src + r * ld);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            acc[2 * e] += (double)bf16_lo(w[e]);
            acc[2 * e + 1] += (double)bf16_hi(w[e]);
        }
    }
    __shared__ double part[kRows][D + 1];
#pragma unroll
    for (int e = 0; e < 8; ++e) part[row][col * 8 + e] = acc[e];
    __syncthreads();
    if (threadIdx.x < D) {
        double t = 0.0;
#pragma unroll
        for (int r = 0; r < kRows; ++r) t += part[r][threadIdx.x];
        out[(b * H + h) * D + threadIdx.x] = (float)(t / (double)count);
    }
}

constexpr int kTile = 64;   // query rows (and key blocks) per score tile
constexpr int kDepth = 16;  // channels per step

// score[unit][i][j] = sum_d qm[i, h, d] * km[j, h, d] in 64 bits, one unit
// being 64 query blocks of a head.  256 threads, 4 x 4 scores each.
__global__ void __launch_bounds__(256) score_kernel(const float* __restrict__ qm, const float* __restrict__ km,
                                                    int nq, int64_t nk, int H, int D, int tiles, int64_t unit0,
                                                    double* __restrict__ score) {
    __shared__ double qs[kDepth][kTile + 1];
    __shared__ double ks[kDepth][kTile + 1];
    const int64_t unit = unit0 + blockIdx.y;
    const int h = (int)(unit / tiles);
    const int64_t i0 = (unit % tiles) * kTile;
    const int64_t j0 = (int64_t)blockIdx.x * kTile;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    double acc[4][4] = {};
    for (int d0 = 0; d0 < D; d0 += kDepth) {
        for (int e = threadIdx.x; e < kTile * kDepth; e += 256) {
            const int d = e % kDepth, r = e / kDepth;
            qs[d][r] = i0 + r < nq ? (double)qm[((i0 + r) * H + h) * D + d0 + d] : 0.0;
            ks[d][r] = j0 + r < nk ? (double)km[((j0 + r) * H + h) * D + d0 + d] : 0.0;
        }
        __syncthreads();
#pragma unroll
        for (int d = 0; d < kDepth; ++d) {
            double a[4], b[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                a[e] = qs[d][ty + 16 * e];
                b[e] = ks[d][tx + 16 * e];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int f = 0; f < 4; ++f) acc[e][f] = fma(a[e], b[f], acc[e][f]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            const int64_t j = j0 + tx + 16 * f;
            if (j < nk) score[((int64_t)blockIdx.y * kTile + ty + 16 * e) * nk + j] = acc[e][f];
        }
}

// Unsigned key in the order of the scores: NaN lowest, -0 with +0.
__device__ __forceinline__ uint64_t sort_key(double s) {
    if (s != s) return 0;
    const uint64_t u = (uint64_t)__double_as_longlong(s + 0.0);
    return u >> 63 ? ~u : u | (1ull << 63);
}

// One CTA per (head, query block): radix selection of the topk-th largest key,
// eight bits a pass, then the chosen indices in ascending order.
__global__ void __launch_bounds__(kThreads) topk_kernel(const double* __restrict__ score, int nq, int64_t nk, int tiles,
                                                        int64_t unit0, int topk, int32_t* __restrict__ blocks) {
    __shared__ int hist[256];
    __shared__ uint64_t s_prefix;
    __shared__ int s_want;
    __shared__ int warp_n[kThreads / 32][2];
    const int64_t unit = unit0 + blockIdx.x / kTile;
    const int h = (int)(unit / tiles);
    const int64_t i = (unit % tiles) * kTile + blockIdx.x % kTile;
    if (i >= nq) return;
    const double* row = score + (int64_t)blockIdx.x * nk;
    int32_t* out = blocks + ((int64_t)h * nq + i) * topk;
    uint64_t prefix = 0;
    int want = topk;  // how many are still to be taken among the keys with this prefix
    for (int shift = 56; shift >= 0; shift -= 8) {
        hist[threadIdx.x] = 0;
        __syncthreads();
        for (int64_t j = threadIdx.x; j < nk; j += kThreads) {
            const uint64_t key = sort_key(row[j]);
            if (shift == 56 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(key >> shift) & 255], 1);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            int left = want, digit = 255;
            while (digit > 0 && hist[digit] < left) left -= hist[digit--];
            s_prefix = prefix | ((uint64_t)digit << shift);
            s_want = left;
        }
        __syncthreads();
        prefix = s_prefix;
        want = s_want;
        __syncthreads();
    }
    // every key above `prefix` is taken, and the first `want` equal to it
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int above = 0, equal = 0;  // so far, before this round's
    for (int64_t j0 = 0; j0 < nk; j0 += kThreads) {
        const int64_t j = j0 + threadIdx.x;
        const uint64_t key = j < nk ? sort_key(row[j]) : 0;
        const bool gt = j < nk && key > prefix, eq = j < nk && key == prefix;
        const uint32_t mg = __ballot_sync(0xFFFFFFFFu, gt), me = __ballot_sync(0xFFFFFFFFu, eq);
        if (lane == 0) {
            warp_n[warp][0] = __popc(mg);
            warp_n[warp][1] = __popc(me);
        }
        __syncthreads();
        int g = above, q = equal;
        for (int w = 0; w < kThreads / 32; ++w) {
            if (w < warp) {
                g += warp_n[w][0];
                q += warp_n[w][1];
            }
            above += warp_n[w][0];
            equal += warp_n[w][1];
        }
        const uint32_t below = (1u << lane) - 1u;
        g += __popc(mg & below);
        q += __popc(me & below);
        if (gt || (eq && q < want)) out[g + min(q, want)] = (int32_t)j;
        __syncthreads();
    }
}

}  // namespace sel
}  // namespace h3b

using namespace h3b;

extern "C" int h3b_block_means(const void* x, int64_t ld, int64_t hs, int64_t S, int64_t H, int64_t D, int64_t rows,
                               float* out, void* stream) {
    H3B_REQUIRE(D == 64 || D == 128, "h3b_block_means: head_dim=%lld must be 64 or 128", (long long)D);
    H3B_REQUIRE(S >= 0 && H > 0 && H <= 65535 && (rows == 64 || rows == 128),
                "h3b_block_means: S=%lld heads=%lld rows=%lld (64 or 128) out of range", (long long)S, (long long)H,
                (long long)rows);
    if (S == 0) return H3B_OK;
    H3B_REQUIRE(x && out && aligned(x, 16) && ld % 8 == 0 && hs % 8 == 0,
                "h3b_block_means: x / out NULL, x not 16-byte aligned or strides not multiples of 8 elements");
    H3B_REQUIRE(cdiv(S, rows) * H < (1ll << 31), "h3b_block_means: too many blocks");
    const unsigned grid = (unsigned)(cdiv(S, rows) * H);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const uint16_t* p = static_cast<const uint16_t*>(x);
    if (D == 128) sel::means_kernel<128><<<grid, sel::kThreads, 0, s>>>(p, ld, hs, S, (int)H, (int)rows, out);
    else sel::means_kernel<64><<<grid, sel::kThreads, 0, s>>>(p, ld, hs, S, (int)H, (int)rows, out);
    H3B_CUDA_TRY(cudaGetLastError());
    return H3B_OK;
}

extern "C" int64_t h3b_select_blocks_workspace(int64_t nq, int64_t nk, int64_t H) {
    if (nq <= 0 || nk <= 0 || H <= 0) return 0;
    const int64_t unit = sel::kTile * nk * 8, units = cdiv(nq, sel::kTile) * H;
    const int64_t most = (256ll << 20) / unit;
    return unit * (units < most ? units : (most > 0 ? most : 1));
}

extern "C" int h3b_select_blocks(const float* qm, const float* km, int64_t nq, int64_t nk, int64_t H, int64_t D,
                                 int64_t topk, int32_t* blocks, void* workspace, int64_t workspace_bytes,
                                 void* stream) {
    H3B_REQUIRE(D == 64 || D == 128, "h3b_select_blocks: head_dim=%lld must be 64 or 128", (long long)D);
    H3B_REQUIRE(nq >= 0 && nk >= 0 && H > 0 && H <= 65535 && nq < (1ll << 31) - 64 && nk < (1ll << 31) - 64,
                "h3b_select_blocks: nq=%lld nk=%lld heads=%lld out of range", (long long)nq, (long long)nk, (long long)H);
    H3B_REQUIRE(topk >= 0 && topk <= nk, "h3b_select_blocks: topk=%lld must lie in [0, %lld]", (long long)topk,
                (long long)nk);
    if (nq == 0 || topk == 0) return H3B_OK;
    H3B_REQUIRE(qm && km && blocks && workspace && aligned(workspace, 8), "h3b_select_blocks: NULL pointer");
    const int64_t unit = sel::kTile * nk * 8;
    const int tiles = (int)cdiv(nq, sel::kTile);
    const int64_t units = (int64_t)tiles * H;
    int64_t per = workspace_bytes / unit;
    H3B_REQUIRE(per > 0, "h3b_select_blocks: the workspace of %lld bytes holds less than one unit of %lld",
                (long long)workspace_bytes, (long long)unit);
    if (per > 65535) per = 65535;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    for (int64_t u = 0; u < units; u += per) {
        const int64_t m = units - u < per ? units - u : per;
        const dim3 grid((unsigned)cdiv(nk, sel::kTile), (unsigned)m);
        double* score = static_cast<double*>(workspace);
        sel::score_kernel<<<grid, 256, 0, s>>>(qm, km, (int)nq, nk, (int)H, (int)D, tiles, u, score);
        sel::topk_kernel<<<(unsigned)(m * sel::kTile), sel::kThreads, 0, s>>>(score, (int)nq, nk, tiles, u, (int)topk,
                                                                             blocks);
    }
    H3B_CUDA_TRY(cudaGetLastError());
    return H3B_OK;
}
