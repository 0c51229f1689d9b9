// Selection of key blocks for block-sparse attention: the means of blocks of
// rows, the products of the means, and the top-k of each (head, query block).
//
// A selection hangs on differences between scores, so sums are held in 64 bits:
// means are rounded once to 32 bits; scores are sums of exact products; equal
// scores go to the lowest index.  A NaN score ranks below every number, -0
// equals +0.  Where a sum fits 53 bits its order does not matter: a block of 128
// rows whose nonzero values lie within a factor of 2^38 (8 + 38 bits and 7 for
// the carries) has the same mean in any order.  Beyond, and in the scores, an
// order may change the last bits of the 64; each kernel's own is fixed, but
// score_kernel and score_few_kernel have different ones, and so may rank blocks
// differently whose scores are equal but for that.
#include "quant_common.cuh"

namespace h3b {
namespace sel {

constexpr int kThreads = 256;

// bf16 -> fp64 times 2^-896 without a conversion instruction (of which an SM does
// too few to keep up with its reads): the exponent and mantissa moved into place,
// which holds for subnormal values as well; infinities and NaNs need the exact
// conversion.  Sums of such values are the exact conversions' sums scaled.
__device__ __forceinline__ double scaled_lo(uint32_t w) {
    return __hiloint2double(((int)(w << 16) >> 3) & 0x8FFFFFFF, 0);
}
__device__ __forceinline__ double scaled_hi(uint32_t w) { return __hiloint2double(((int)w >> 3) & 0x8FFFE000, 0); }
constexpr double kDown = 0x1p-896, kUp = 0x1p896;

struct Means {
    const uint16_t* x;  // [S, H, D]
    int64_t ld, hs, S;
    float* out;  // [nb, H, D]
    int64_t ctas;  // blocks x heads
};

// More bytes in flight for its registers than 256 threads with half the rows each.
constexpr int kMeanThreads = 128;

// mean over the rows of a block of x -> fp32, one CTA per (block, head); 8
// channels a thread, kMeanThreads / (D / 8) row lanes.  Bound by its reads; a whole
// block's loads are in flight before the first is used (128000 rows of 5 heads,
// keys and queries: 64 us, 5.2 TB/s).
template <int D, int ROWS>
__device__ __forceinline__ void block_mean(const Means& a, int H, int64_t cta) {
    constexpr int kCols = D / 8;
    constexpr int kRows = kMeanThreads / kCols;
    constexpr int kLoads = ROWS / kRows;
    constexpr int kWarps = kMeanThreads / 32;
    const int64_t b = (int64_t)((uint32_t)cta / (uint32_t)H);
    const int h = (int)((uint32_t)cta - (uint32_t)b * (uint32_t)H);
    const int col = threadIdx.x % kCols, row = threadIdx.x / kCols;
    const int count = (int)min((int64_t)ROWS, a.S - b * ROWS);
    const uint16_t* src = a.x + (b * ROWS + row) * a.ld + h * a.hs + col * 8;
    uint4 v[kLoads];
#pragma unroll
    for (int p = 0; p < kLoads; ++p) {
        v[p] = make_uint4(0, 0, 0, 0);
        if (row + p * kRows < count) v[p] = __ldcs(reinterpret_cast<const uint4*>(src + (int64_t)p * kRows * a.ld));
    }
    double acc[8] = {};
    uint32_t top = 0;  // largest |x| of the low and of the high halves
#pragma unroll
    for (int p = 0; p < kLoads; ++p) top = absmax_bits8(v[p], top);
    if (max(top & 0xFFFFu, top >> 16) < 0x7F80u) {
#pragma unroll
        for (int p = 0; p < kLoads; ++p) {
            const uint32_t w[4] = {v[p].x, v[p].y, v[p].z, v[p].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                acc[2 * e] += scaled_lo(w[e]);
                acc[2 * e + 1] += scaled_hi(w[e]);
            }
        }
    } else {
#pragma unroll
        for (int p = 0; p < kLoads; ++p) {
            const uint32_t w[4] = {v[p].x, v[p].y, v[p].z, v[p].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                acc[2 * e] += (double)bf16_lo(w[e]) * kDown;
                acc[2 * e + 1] += (double)bf16_hi(w[e]) * kDown;
            }
        }
    }
    // the row lanes of a warp, then the warps
    __shared__ double part[kWarps][D];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
#pragma unroll
        for (int off = kCols; off < 32; off <<= 1) acc[e] += __shfl_xor_sync(0xFFFFFFFFu, acc[e], off);
        if (threadIdx.x % 32 < kCols) part[threadIdx.x / 32][col * 8 + e] = acc[e];
    }
    __syncthreads();
    for (int ch = threadIdx.x; ch < D; ch += kMeanThreads) {
        double t = 0.0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) t += part[w][ch];
        a.out[(b * H + h) * D + ch] = (float)(t * kUp / (double)count);
    }
}

// Blocks of 64 rows of one tensor and of 128 rows of another (either may have none).
template <int D>
__global__ void __launch_bounds__(kMeanThreads) means_kernel(const __grid_constant__ Means by64,
                                                         const __grid_constant__ Means by128, int H) {
    if (blockIdx.x < by64.ctas) block_mean<D, 64>(by64, H, blockIdx.x);
    else block_mean<D, 128>(by128, H, blockIdx.x - by64.ctas);
}

static int launch_means(const Means& by64, const Means& by128, int64_t H, int64_t D, cudaStream_t s) {
    const unsigned grid = (unsigned)(by64.ctas + by128.ctas);
    if (grid == 0) return H3B_OK;
    if (D == 128) means_kernel<128><<<grid, kMeanThreads, 0, s>>>(by64, by128, (int)H);
    else means_kernel<64><<<grid, kMeanThreads, 0, s>>>(by64, by128, (int)H);
    H3B_CUDA_TRY(cudaGetLastError());
    return H3B_OK;
}

static int check_means(const char* who, const void* x, int64_t ld, int64_t hs, int64_t S, int64_t H, int64_t rows,
                       float* out, Means* m) {
    *m = Means{static_cast<const uint16_t*>(x), ld, hs, S, out, cdiv(S, rows) * H};
    if (S == 0) return H3B_OK;
    H3B_REQUIRE(x && out && aligned(x, 16) && ld > 0 && hs > 0 && ld % 8 == 0 && hs % 8 == 0,
                "%s: x / out NULL, x not 16-byte aligned or strides not positive multiples of 8 elements", who);
    H3B_REQUIRE(m->ctas < (1ll << 30), "%s: too many blocks", who);
    return H3B_OK;
}

constexpr int kTile = 64;  // query rows (and key blocks) per score tile
constexpr int kFew = 4;    // query blocks up to which the scores are plain products

// score[unit][i][j] = sum_d qm[i, h, d] * km[j, h, d] in 64 bits, one unit
// being 64 query blocks of a head.  Four warps a tile of T x T by mma.sync m8n8k4
// in fp64; both operands lie in shared memory as fp32, their whole depth at once.
// Bound by the fp64 products with T = 64 (1000 x 2000 blocks of 5 heads: 109 us,
// 75 at the fp64 rate); T = 32 where there are too few such
// tiles for the SMs (33 x 65 blocks of 40 heads).
template <int D, int T>
__global__ void __launch_bounds__(128) score_kernel(const float* __restrict__ qm, const float* __restrict__ km, int nq,
                                                    int64_t nk, int H, int tiles, int64_t unit0,
                                                    double* __restrict__ score) {
    constexpr int kLd = D + 4;  // 8 rows x 4 channels of an operand meet 32 banks
    extern __shared__ __align__(16) float tile[];
    float *qs = tile, *ks = tile + T * kLd;
    constexpr int kSub = kTile / T;  // tiles down a unit
    const int64_t unit = unit0 + blockIdx.y / kSub;
    const int sub = blockIdx.y % kSub * T;
    const int h = (int)(unit / tiles);
    const int64_t i0 = (unit % tiles) * kTile + sub, j0 = (int64_t)blockIdx.x * T;
    if (i0 >= nq) return;
    for (int e = threadIdx.x; e < T * (D / 4); e += 128) {
        const int r = e / (D / 4), d = e % (D / 4) * 4;
        float4 x = make_float4(0, 0, 0, 0), y = x;
        if (i0 + r < nq) x = *reinterpret_cast<const float4*>(qm + ((i0 + r) * H + h) * D + d);
        if (j0 + r < nk) y = *reinterpret_cast<const float4*>(km + ((j0 + r) * H + h) * D + d);
        *reinterpret_cast<float4*>(qs + r * kLd + d) = x;
        *reinterpret_cast<float4*>(ks + r * kLd + d) = y;
    }
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int E = T / 16;  // products of 8 x 8 along a warp's side
    const int wi = (warp >> 1) * (T / 2), wj = (warp & 1) * (T / 2);
    const float* qa = qs + (wi + (lane >> 2)) * kLd + (lane & 3);
    const float* ka = ks + (wj + (lane >> 2)) * kLd + (lane & 3);
    double acc[E][E][2] = {};
#pragma unroll 4
    for (int d = 0; d < D; d += 4) {
        double x[E], y[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            x[e] = (double)qa[e * 8 * kLd + d];
            y[e] = (double)ka[e * 8 * kLd + d];
        }
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int f = 0; f < E; ++f)
                asm("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};"
                    : "+d"(acc[e][f][0]), "+d"(acc[e][f][1])
                    : "d"(x[e]), "d"(y[f]));
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
        for (int f = 0; f < E; ++f)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int64_t j = j0 + wj + 8 * f + 2 * (lane & 3) + k;
                if (j < nk) score[((int64_t)(blockIdx.y / kSub) * kTile + sub + wi + 8 * e + (lane >> 2)) * nk + j] = acc[e][f][k];
            }
}

// The same for up to kFew query blocks: one warp a key block, so that the means
// of the keys are read once at full width.
template <int D>
__global__ void __launch_bounds__(kThreads) score_few_kernel(const float* __restrict__ qm, const float* __restrict__ km,
                                                             int nq, int64_t nk, int H, int64_t unit0,
                                                             double* __restrict__ score) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31;
    const int64_t j = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    const int h = (int)(unit0 + blockIdx.y);
    if (j >= nk) return;
    double y[E];
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = (double)km[(j * H + h) * D + lane + 32 * e];
    for (int i = 0; i < nq; ++i) {
        double t = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) t = fma((double)qm[((int64_t)i * H + h) * D + lane + 32 * e], y[e], t);
#pragma unroll
        for (int off = 16; off; off >>= 1) t += __shfl_xor_sync(0xFFFFFFFFu, t, off);
        if (lane == 0) score[((int64_t)blockIdx.y * kTile + i) * nk + j] = t;
    }
}

// Unsigned key in the order of the scores: NaN lowest, -0 with +0.
__device__ __forceinline__ uint64_t sort_key(double s) {
    if (s != s) return 0;
    const uint64_t u = (uint64_t)__double_as_longlong(s + 0.0);
    return u >> 63 ? ~u : u | (1ull << 63);
}

// One CTA per (head, query block): radix selection of the topk-th largest key,
// eight bits a pass until all keys that share the digits so far are taken, then
// the chosen indices in ascending order.  HELD keys a thread (every kThreads-th)
// stay in registers; with HELD 0 all are read again every pass.  Bound by the
// passes' barriers (5000 rows of 2000 keys: 99 us).
template <int HELD>
__global__ void __launch_bounds__(kThreads, HELD <= 8 ? 6 : 4) topk_kernel(const double* __restrict__ score, int nq, int64_t nk, int tiles,
                                                        int64_t unit0, int topk, int per, int32_t* __restrict__ blocks) {
    constexpr int kWarps = kThreads / 32;
    __shared__ int hist[256];
    __shared__ int s_digit, s_left, s_count;
    __shared__ int taken[2][(HELD > 0 ? HELD : 1) * kWarps];  // above the prefix, with it: by round and warp
    const int64_t unit = unit0 + blockIdx.x / per;
    const int h = (int)(unit / tiles), r = blockIdx.x % per;  // `per` rows of a unit are in the launch
    const int64_t i = (unit % tiles) * kTile + r;
    if (i >= nq) return;
    const double* row = score + ((int64_t)(blockIdx.x / per) * kTile + r) * nk;
    int32_t* out = blocks + ((int64_t)h * nq + i) * topk;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (topk == nk) {
        for (int64_t j = threadIdx.x; j < nk; j += kThreads) out[j] = (int32_t)j;
        return;
    }
    const int rounds = (int)((nk + kThreads - 1) / kThreads);
    uint64_t held[HELD > 0 ? HELD : 1];
    if constexpr (HELD > 0) {
#pragma unroll
        for (int t = 0; t < HELD; ++t) {
            const int64_t j = threadIdx.x + t * kThreads;
            held[t] = j < nk ? sort_key(row[j]) : 0;
        }
    }
    auto each = [&](auto&& f) {
        if constexpr (HELD > 0) {
#pragma unroll
            for (int t = 0; t < HELD; ++t) f(threadIdx.x + t * kThreads, held[t], t);
        } else {
            for (int t = 0; t < rounds; ++t) {
                const int64_t j = threadIdx.x + (int64_t)t * kThreads;
                f(j, j < nk ? sort_key(row[j]) : 0, t);
            }
        }
    };
    uint64_t prefix = 0;
    int want = topk;  // how many are still to be taken among the keys with this prefix
    int shift = 56;
    for (;; shift -= 8) {
        hist[threadIdx.x] = 0;
        __syncthreads();
        each([&](int64_t j, uint64_t key, int) {
            const bool in = j < nk && (shift == 56 || (key >> (shift + 8)) == (prefix >> (shift + 8)));
            const uint32_t digit = in ? (uint32_t)(key >> shift) & 255u : 256u;
            if (shift >= 48) {
                // most keys share their exponent's digits: one addition for a warp's equal ones
                const uint32_t same = __match_any_sync(0xFFFFFFFFu, digit);
                if (in && lane == __ffs(same) - 1) atomicAdd(&hist[digit], __popc(same));
            } else if (in) {
                atomicAdd(&hist[digit], 1);
            }
        });
        __syncthreads();
        if (warp == 0) {
            // digits 255 - 8 lane downwards: the one in which the want-th largest lies
            int n[8], sum = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                n[e] = hist[255 - 8 * lane - e];
                sum += n[e];
            }
            int above = sum;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int y = __shfl_up_sync(0xFFFFFFFFu, above, off);
                if (lane >= off) above += y;
            }
            above -= sum;  // keys with a larger digit than this lane's
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (above < want && want <= above + n[e]) {
                    s_digit = 255 - 8 * lane - e;
                    s_left = want - above;
                    s_count = n[e];
                }
                above += n[e];
            }
        }
        __syncthreads();
        prefix |= (uint64_t)s_digit << shift;
        want = s_left;
        const bool all = s_count == want;
        __syncthreads();
        if (all || shift == 0) break;
    }
    // every key above the prefix is taken, and the first `want` that have it
    const uint32_t below = (1u << lane) - 1u;
    const uint64_t bar = prefix >> shift;
    if constexpr (HELD > 0) {
        // counts of every round and warp, their sum before each, then the places
        each([&](int64_t j, uint64_t key, int t) {
            const uint64_t head = key >> shift;
            const uint32_t mg = __ballot_sync(0xFFFFFFFFu, j < nk && head > bar),
                           me = __ballot_sync(0xFFFFFFFFu, j < nk && head == bar);
            if (lane == 0) {
                taken[0][t * kWarps + warp] = __popc(mg);
                taken[1][t * kWarps + warp] = __popc(me);
            }
        });
        __syncthreads();
        if (warp < 2) {
            constexpr int kEach = (HELD * kWarps + 31) / 32;
            int n[kEach], sum = 0;
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                const int at = lane * kEach + e;
                n[e] = at < HELD * kWarps ? taken[warp][at] : 0;
                sum += n[e];
            }
            int before = sum;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int y = __shfl_up_sync(0xFFFFFFFFu, before, off);
                if (lane >= off) before += y;
            }
            before -= sum;
            __syncwarp();
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                const int at = lane * kEach + e;
                if (at < HELD * kWarps) taken[warp][at] = before;
                before += n[e];
            }
        }
        __syncthreads();
        each([&](int64_t j, uint64_t key, int t) {
            const uint64_t head = key >> shift;
            const bool gt = j < nk && head > bar, eq = j < nk && head == bar;
            const uint32_t mg = __ballot_sync(0xFFFFFFFFu, gt), me = __ballot_sync(0xFFFFFFFFu, eq);
            const int g = taken[0][t * kWarps + warp] + __popc(mg & below), q = taken[1][t * kWarps + warp] + __popc(me & below);
            if (gt || (eq && q < want)) out[g + min(q, want)] = (int32_t)j;
        });
    } else {
        int above = 0, equal = 0;  // so far, before this round's
        each([&](int64_t j, uint64_t key, int) {
            const uint64_t head = key >> shift;
            const bool gt = j < nk && head > bar, eq = j < nk && head == bar;
            const uint32_t mg = __ballot_sync(0xFFFFFFFFu, gt), me = __ballot_sync(0xFFFFFFFFu, eq);
            if (lane == 0) {
                taken[0][warp] = __popc(mg);
                taken[1][warp] = __popc(me);
            }
            __syncthreads();
            int g = above, q = equal;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                if (w < warp) {
                    g += taken[0][w];
                    q += taken[1][w];
                }
                above += taken[0][w];
                equal += taken[1][w];
            }
            g += __popc(mg & below);
            q += __popc(me & below);
            if (gt || (eq && q < want)) out[g + min(q, want)] = (int32_t)j;
            __syncthreads();
        });
    }
}

template <int D>
static int scores(const float* qm, const float* km, int nq, int64_t nk, int H, int tiles, int64_t unit, int64_t units,
                  double* score, cudaStream_t s) {
    if (nq <= kFew) {
        const dim3 grid((unsigned)cdiv(nk, kThreads / 32), (unsigned)units);
        score_few_kernel<D><<<grid, kThreads, 0, s>>>(qm, km, nq, nk, H, unit, score);
    } else {
        const int64_t big = cdiv(nk, kTile) * units;
        constexpr int smem64 = 2 * 64 * (D + 4) * 4, smem32 = 2 * 32 * (D + 4) * 4;
        if (big >= 2 * 148) {  // two a SM
            H3B_CUDA_TRY(cudaFuncSetAttribute(score_kernel<D, 64>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem64));
            score_kernel<D, 64><<<dim3((unsigned)cdiv(nk, 64), (unsigned)units), 128, smem64, s>>>(qm, km, nq, nk, H, tiles,
                                                                                                unit, score);
        } else {
            score_kernel<D, 32><<<dim3((unsigned)cdiv(nk, 32), (unsigned)(2 * units)), 128, smem32, s>>>(
                qm, km, nq, nk, H, tiles, unit, score);
        }
    }
    H3B_CUDA_TRY(cudaGetLastError());
    return H3B_OK;
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
    sel::Means m, none{};
    if (int rc = sel::check_means("h3b_block_means", x, ld, hs, S, H, rows, out, &m)) return rc;
    return rows == 64 ? sel::launch_means(m, none, H, D, static_cast<cudaStream_t>(stream))
                      : sel::launch_means(none, m, H, D, static_cast<cudaStream_t>(stream));
}

// Means of 64 keys and of 128 query rows in one launch (sparse.cu).
namespace h3b {
int sparse_means(const void* k, int64_t k_ld, int64_t k_hs, int64_t Sk, float* km, const void* q, int64_t q_ld,
                 int64_t q_hs, int64_t Sq, float* qm, int64_t H, int64_t D, cudaStream_t s) {
    sel::Means a{}, b;
    if (km) {
        if (int rc = sel::check_means("h3b_sparse_attn", k, k_ld, k_hs, Sk, H, 64, km, &a)) return rc;
    }
    if (int rc = sel::check_means("h3b_sparse_attn", q, q_ld, q_hs, Sq, H, 128, qm, &b)) return rc;
    return sel::launch_means(a, b, H, D, s);
}
}  // namespace h3b

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
    H3B_REQUIRE(qm && km && blocks && workspace && aligned(workspace, 8) && aligned(qm, 16) && aligned(km, 16),
                "h3b_select_blocks: NULL pointer, or means not 16-byte aligned");
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
        double* score = static_cast<double*>(workspace);
        if (int rc = D == 128 ? sel::scores<128>(qm, km, (int)nq, nk, (int)H, tiles, u, m, score, s)
                              : sel::scores<64>(qm, km, (int)nq, nk, (int)H, tiles, u, m, score, s))
            return rc;
        const int held = (int)cdiv(nk, sel::kThreads), per = nq < sel::kTile ? (int)nq : sel::kTile;
        const unsigned rows = (unsigned)(m * per);
        if (held == 1)
            sel::topk_kernel<1><<<rows, sel::kThreads, 0, s>>>(score, (int)nq, nk, tiles, u, (int)topk, per, blocks);
        else if (held <= 4)
            sel::topk_kernel<4><<<rows, sel::kThreads, 0, s>>>(score, (int)nq, nk, tiles, u, (int)topk, per, blocks);
        else if (held <= 8)
            sel::topk_kernel<8><<<rows, sel::kThreads, 0, s>>>(score, (int)nq, nk, tiles, u, (int)topk, per, blocks);
        else if (held <= 16)
            sel::topk_kernel<16><<<rows, sel::kThreads, 0, s>>>(score, (int)nq, nk, tiles, u, (int)topk, per, blocks);
        else
            sel::topk_kernel<0><<<rows, sel::kThreads, 0, s>>>(score, (int)nq, nk, tiles, u, (int)topk, per, blocks);
    }
    H3B_CUDA_TRY(cudaGetLastError());
    return H3B_OK;
}
