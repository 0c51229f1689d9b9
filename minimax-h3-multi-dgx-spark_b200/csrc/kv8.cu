// Key/value cache held in 8 bits: quantise while writing, and read back.
//
// codes [H, cap, D] int8, scales [H, cap / 64] fp32, K and V apart: the tokens
// of one head lie together, so a tile of any 128 tokens that the attention
// takes is one contiguous run, and a block of 64 tokens of a head (what shares
// a scale) is 64 * D consecutive bytes.
//
//   scale = max |x| / 127 over the block's new tokens (IEEE division), or the
//           block's older scale where older tokens stay and it is larger in
//           magnitude (a cache that was not written here may have negative
//           ones: the sign stays, as do the codes that go with it);
//   code  = clamp(rint_half_even(x / scale), -127, 127), 0 for scale 0;
//   codes that stay are requantised, rint(code * (old / scale)), if the scale grew.
// A non-finite x makes the scale non-finite and the block's codes 0, so
// everything read from it is NaN.  Maxima run on the bit patterns of |x|,
// which order NaN above infinity above the numbers.
#include "quant_common.cuh"

namespace h3b {
namespace kv8 {

constexpr int kBlock = 64;  // tokens per scale
constexpr int kThreads = 256;
constexpr int kWriteThreads = 128;

struct WriteArgs {
    const uint16_t* x[2];  // k, v: [n, H, D], strides in elements
    int64_t ld[2], hs[2];
    int8_t* codes[2];
    float* scales[2];
    int64_t cap, start, n;
    int H;
};

__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
    return (uint32_t)(a & 255) | ((uint32_t)(b & 255) << 8) | ((uint32_t)(c & 255) << 16) | ((uint32_t)(d & 255) << 24);
}

// One CTA per block of 64 tokens and head (blockIdx.x) and per K / V
// (blockIdx.y).  A thread holds 8 consecutive channels of PASSES tokens in
// registers between the maximum and the division, so x is read once.  Bound by
// HBM in principle (x once, codes once); 128 threads with twice the tokens each
// rather than 256, because what a thread does besides its tokens counts here
// (33024 tokens of 40 heads: 193 us instead of 295, 5.3 TB/s).
template <int D>
__global__ void __launch_bounds__(kWriteThreads) write_kernel(const __grid_constant__ WriteArgs a) {
    constexpr int kCols = D / 8;                  // threads along the channels
    constexpr int kRows = kWriteThreads / kCols;  // tokens per pass
    constexpr int kPasses = kBlock / kRows;
    const int which = blockIdx.y;
    const unsigned nth = blockIdx.x / (unsigned)a.H;
    const int h = (int)(blockIdx.x - nth * (unsigned)a.H);
    const int64_t b = a.start / kBlock + nth;
    // new tokens are rows first .. last - 1 of the block, older ones lie before
    const int first = (int)max(a.start - b * kBlock, (int64_t)0);
    const int last = (int)min(a.start + a.n - b * kBlock, (int64_t)kBlock);
    const int col = threadIdx.x % kCols, row = threadIdx.x / kCols;
    int8_t* codes = a.codes[which] + ((int64_t)h * a.cap + b * kBlock + row) * D + col * 8;
    float* scale = a.scales[which] + (int64_t)h * (a.cap / kBlock) + b;
    const int64_t ld = a.ld[which];
    const uint16_t* x = a.x[which] + (b * kBlock - a.start + row) * ld + h * a.hs[which] + col * 8;

    uint4 v[kPasses];
    uint32_t pair = 0;  // maxima of the low and of the high halves' bits
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
        const int r = row + p * kRows;
        v[p] = make_uint4(0, 0, 0, 0);
        if (r >= first && r < last) v[p] = __ldcs(reinterpret_cast<const uint4*>(x + p * kRows * ld));
    }
    const bool stays = first > 0;  // older tokens in this block
    const float older = stays ? *scale : 0.0f;
#pragma unroll
    for (int p = 0; p < kPasses; ++p) pair = absmax_bits8(v[p], pair);
    __shared__ uint32_t tops[kWriteThreads / 32];
    uint32_t top = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(fold_absmax_bits(pair)));
    if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWriteThreads / 32; ++w) top = max(top, tops[w]);
    // a NaN's quotient is a NaN: the order of the bit patterns still holds below
    float s = __fdiv_rn(__uint_as_float(top), 127.0f);
    if ((__float_as_uint(older) & 0x7FFFFFFFu) > (__float_as_uint(s) & 0x7FFFFFFFu)) s = older;
    const bool live = s != 0.0f && fabsf(s) < __int_as_float(0x7F800000);
    const float inverse = live ? __frcp_rn(s) : 0.0f;
    const bool grew = stays && __float_as_uint(s) != __float_as_uint(older);
    const float ratio = grew && live ? __fdiv_rn(older, s) : 0.0f;
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
        const int r = row + p * kRows;
        uint2* dst = reinterpret_cast<uint2*>(codes + p * kRows * D);
        if (r >= first && r < last) {
            float f[8];
            unpack8(v[p], f);
            // (the scale's magnitude is the block's absmax / 127 or larger, so no code leaves [-127, 127])
            *dst = live ? quant8(f, s, inverse) : make_uint2(0u, 0u);
        } else if (grew && r < first) {
            const uint2 old = *dst;
            int c[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int8_t q = (int8_t)(((e < 4 ? old.x : old.y) >> (8 * (e & 3))) & 255u);
                c[e] = (int)rintf(__fmul_rn((float)q, ratio));
            }
            *dst = make_uint2(pack4(c[0], c[1], c[2], c[3]), pack4(c[4], c[5], c[6], c[7]));
        }
    }
    // `older` was read by every thread before the barrier above
    if (threadIdx.x == 0) *scale = s;
}

struct ReadArgs {
    const int8_t* codes[2];
    const float* scales[2];
    void* out[2];  // [n, H, D]
    int64_t cap, start, n;
    int H;
};

// One CTA per block of 64 tokens and head, per K / V; 8 codes a thread and pass.
// Bound by HBM (33024 tokens of 40 heads to bf16: 152 us, 6.7 TB/s).
template <int D, bool F32>
__global__ void __launch_bounds__(kThreads) read_kernel(const __grid_constant__ ReadArgs a) {
    constexpr int kCols = D / 8;
    constexpr int kRows = kThreads / kCols;
    const int which = blockIdx.y;
    const int h = (int)(blockIdx.x % (unsigned)a.H);
    const int64_t b = a.start / kBlock + blockIdx.x / (unsigned)a.H;
    const int col = threadIdx.x % kCols, row = threadIdx.x / kCols;
    const int8_t* codes = a.codes[which] + ((int64_t)h * a.cap + b * kBlock) * D + col * 8;
    const float s = a.scales[which][(int64_t)h * (a.cap / kBlock) + b];
    uint2 v[kBlock / kRows];
#pragma unroll
    for (int p = 0; p < kBlock / kRows; ++p) {
        const int64_t t = b * kBlock + row + p * kRows;
        if (t >= a.start && t < a.start + a.n) v[p] = *reinterpret_cast<const uint2*>(codes + (row + p * kRows) * D);
    }
#pragma unroll
    for (int p = 0; p < kBlock / kRows; ++p) {
        const int64_t t = b * kBlock + row + p * kRows;
        if (t < a.start || t >= a.start + a.n) continue;
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
            f[e] = __fmul_rn((float)(int8_t)(((e < 4 ? v[p].x : v[p].y) >> (8 * (e & 3))) & 255u), s);
        const int64_t at = ((t - a.start) * a.H + h) * D + col * 8;
        if constexpr (F32) {
            float4* o = reinterpret_cast<float4*>(static_cast<float*>(a.out[which]) + at);
            o[0] = make_float4(f[0], f[1], f[2], f[3]);
            o[1] = make_float4(f[4], f[5], f[6], f[7]);
        } else {
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out[which]) + at) =
                make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                           pack_bf16x2(f[6], f[7]));
        }
    }
}

static int check_cache(const char* who, const void* kq, const void* vq, const void* ks, const void* vs, int64_t cap,
                       int64_t start, int64_t n, int64_t H, int64_t D) {
    H3B_REQUIRE(D == 64 || D == 128, "%s: head_dim=%lld must be 64 or 128", who, (long long)D);
    H3B_REQUIRE(H > 0 && H <= 65535 && cap >= 0 && cap % kBlock == 0 && cap <= (1ll << 31),
                "%s: heads=%lld and capacity=%lld (a multiple of %d) out of range", who, (long long)H, (long long)cap,
                kBlock);
    H3B_REQUIRE(start >= 0 && n >= 0 && start <= cap && n <= cap - start,
                "%s: tokens [%lld, %lld) lie outside the capacity %lld", who, (long long)start, (long long)(start + n),
                (long long)cap);
    H3B_REQUIRE(n == 0 || (kq && vq && ks && vs), "%s: NULL cache pointer", who);
    H3B_REQUIRE(aligned(kq, 16) && aligned(vq, 16) && aligned(ks, 4) && aligned(vs, 4),
                "%s: codes must be 16-byte aligned", who);
    const int64_t blocks = (start + n + kBlock - 1) / kBlock - start / kBlock;
    H3B_REQUIRE(blocks * H < (1ll << 31), "%s: too many blocks in one call", who);
    return H3B_OK;
}

}  // namespace kv8
}  // namespace h3b

using namespace h3b;

extern "C" int h3b_kv8_write(const void* k, int64_t k_ld, int64_t k_hs, const void* v, int64_t v_ld, int64_t v_hs,
                             int64_t start, int64_t n, int64_t H, int64_t D, int8_t* kq, int8_t* vq, float* ks,
                             float* vs, int64_t cap, void* stream) {
    if (int rc = kv8::check_cache("h3b_kv8_write", kq, vq, ks, vs, cap, start, n, H, D)) return rc;
    if (n == 0) return H3B_OK;
    H3B_REQUIRE(k && v && aligned(k, 16) && aligned(v, 16), "h3b_kv8_write: k / v NULL or not 16-byte aligned");
    H3B_REQUIRE(k_ld > 0 && k_hs > 0 && v_ld > 0 && v_hs > 0 && k_ld % 8 == 0 && k_hs % 8 == 0 && v_ld % 8 == 0 &&
                    v_hs % 8 == 0,
                "h3b_kv8_write: token and head strides must be positive multiples of 8 elements");
    kv8::WriteArgs a{{static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v)},
                     {k_ld, v_ld}, {k_hs, v_hs}, {kq, vq}, {ks, vs}, cap, start, n, (int)H};
    const int64_t blocks = cdiv(start + n, kv8::kBlock) - start / kv8::kBlock;
    const dim3 grid((unsigned)(blocks * H), 2);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (D == 128) kv8::write_kernel<128><<<grid, kv8::kWriteThreads, 0, s>>>(a);
    else kv8::write_kernel<64><<<grid, kv8::kWriteThreads, 0, s>>>(a);
    H3B_CUDA_TRY(cudaGetLastError());
    return H3B_OK;
}

extern "C" int h3b_kv8_read(const int8_t* kq, const int8_t* vq, const float* ks, const float* vs, int64_t cap,
                            int64_t start, int64_t n, int64_t H, int64_t D, void* k_out, void* v_out, int fp32,
                            void* stream) {
    if (int rc = kv8::check_cache("h3b_kv8_read", kq, vq, ks, vs, cap, start, n, H, D)) return rc;
    if (n == 0) return H3B_OK;
    H3B_REQUIRE(k_out && v_out && aligned(k_out, 16) && aligned(v_out, 16),
                "h3b_kv8_read: outputs NULL or not 16-byte aligned");
    kv8::ReadArgs a{{kq, vq}, {ks, vs}, {k_out, v_out}, cap, start, n, (int)H};
    const int64_t blocks = cdiv(start + n, kv8::kBlock) - start / kv8::kBlock;
    const dim3 grid((unsigned)(blocks * H), 2);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (D == 128 && fp32) kv8::read_kernel<128, true><<<grid, kv8::kThreads, 0, s>>>(a);
    else if (D == 128) kv8::read_kernel<128, false><<<grid, kv8::kThreads, 0, s>>>(a);
    else if (fp32) kv8::read_kernel<64, true><<<grid, kv8::kThreads, 0, s>>>(a);
    else kv8::read_kernel<64, false><<<grid, kv8::kThreads, 0, s>>>(a);
    H3B_CUDA_TRY(cudaGetLastError());
    return H3B_OK;
}
