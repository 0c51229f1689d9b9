// Attention over a key/value cache held in 8 bits, and over selected blocks of
// bf16 keys:  o = softmax(scale * q k^T) v, one pass over the keys with the
// running maximum and sum of the softmax.
#include "common.cuh"

namespace h3b {
namespace attn {

constexpr int kSeg = 64;     // keys per segment: a cache block, or a selected block
constexpr int kQRows = 128;  // query rows that share a selection

struct Args {
    const uint16_t* q;
    int64_t q_ld, q_hs;
    uint16_t* o;
    int64_t o_ld, o_hs;
    int64_t Sq, keys;
    int H;
    float scale;
    // 8-bit cache
    const int8_t* codes[2];
    const float* scales[2];
    int64_t cap;
    // selected blocks of bf16 keys
    const uint16_t* kv[2];
    int64_t kv_ld[2], kv_hs[2];
    const int32_t* blocks;
    int topk;
    int64_t nq;
    int* status;
};

// One warp per (query row, head); each lane holds D / 32 channels.
template <int D, bool CACHE>
__global__ void __launch_bounds__(128) rows_kernel(Args a) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31;
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (id >= a.Sq * a.H) return;
    const int h = (int)(id % a.H);
    const int64_t row = id / a.H;
    float q[E], o[E] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e)
        q[e] = __uint_as_float((uint32_t)a.q[row * a.q_ld + h * a.q_hs + lane * E + e] << 16) * a.scale;
    const int64_t segs = CACHE ? (a.keys + kSeg - 1) / kSeg : a.topk;
    for (int64_t s = 0; s < segs; ++s) {
        int64_t b = s;
        if constexpr (!CACHE) {
            b = a.blocks[((int64_t)h * a.nq + row / kQRows) * a.topk + s];
            if (b < 0 || b * kSeg >= a.keys) {
                if (b != -1 && lane == 0) report(a.status, H3B_STATUS_BAD_INDEX);
                continue;
            }
        }
        float sk = 1.0f, sv = 1.0f;
        if constexpr (CACHE) {
            sk = a.scales[0][(int64_t)h * (a.cap / kSeg) + b];
            sv = a.scales[1][(int64_t)h * (a.cap / kSeg) + b];
        }
        const int n = (int)min((int64_t)kSeg, a.keys - b * kSeg);
        for (int j = 0; j < n; ++j) {
            const int64_t t = b * kSeg + j;
            float k[E], v[E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if constexpr (CACHE) {
                    const int64_t at = ((int64_t)h * a.cap + t) * D + lane * E + e;
                    k[e] = (float)a.codes[0][at];
                    v[e] = (float)a.codes[1][at];
                } else {
                    k[e] = __uint_as_float((uint32_t)a.kv[0][t * a.kv_ld[0] + h * a.kv_hs[0] + lane * E + e] << 16);
                    v[e] = __uint_as_float((uint32_t)a.kv[1][t * a.kv_ld[1] + h * a.kv_hs[1] + lane * E + e] << 16);
                }
            }
            float x = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) x += q[e] * k[e];
#pragma unroll
            for (int off = 16; off; off >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, off);
            x *= sk;
            const float to = fmaxf(m, x), p = expf(x - to), keep = m == to ? 1.0f : expf(m - to);
            m = to;
            l = l * keep + p;
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = o[e] * keep + p * sv * v[e];
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int e = 0; e < E; ++e)
        a.o[row * a.o_ld + h * a.o_hs + lane * E + e] = (uint16_t)f2bf_bits(o[e] * inv);
}

template <bool CACHE>
static int launch(const char* who, Args& a, int64_t D, cudaStream_t s) {
    H3B_REQUIRE(D == 64 || D == 128, "%s: head_dim=%lld must be 64 or 128", who, (long long)D);
    H3B_REQUIRE(a.Sq >= 0 && a.keys >= 0 && a.H > 0 && a.H <= 65535 && a.Sq < (1ll << 31) && a.keys < (1ll << 31),
                "%s: shape out of range (rows=%lld keys=%lld heads=%d)", who, (long long)a.Sq, (long long)a.keys, a.H);
    if (a.Sq == 0) return H3B_OK;
    H3B_REQUIRE(a.q && a.o && aligned(a.q, 16) && aligned(a.o, 16), "%s: q / o NULL or not 16-byte aligned", who);
    H3B_REQUIRE(a.q_ld % 8 == 0 && a.q_hs % 8 == 0 && a.o_ld % 8 == 0 && a.o_hs % 8 == 0,
                "%s: strides must be multiples of 8 elements", who);
    DeviceStatus ds;
    if (int rc = device_status(&ds)) return rc;
    a.status = ds.word;
    const unsigned grid = (unsigned)cdiv(a.Sq * a.H, 4);
    if (D == 128) rows_kernel<128, CACHE><<<grid, 128, 0, s>>>(a);
    else rows_kernel<64, CACHE><<<grid, 128, 0, s>>>(a);
    H3B_CUDA_TRY(cudaGetLastError());
    return H3B_OK;
}

}  // namespace attn
}  // namespace h3b

using namespace h3b;

extern "C" int h3b_kv8_attn(const void* q, int64_t q_ld, int64_t q_hs, int64_t Sq, int64_t H, int64_t D,
                            const int8_t* kq, const int8_t* vq, const float* ks, const float* vs, int64_t cap,
                            int64_t length, float scale, void* o, int64_t o_ld, int64_t o_hs, void* stream) {
    H3B_REQUIRE(cap >= 0 && cap % attn::kSeg == 0 && length >= 0 && length <= cap,
                "h3b_kv8_attn: length=%lld must lie within the capacity %lld (a multiple of %d)", (long long)length,
                (long long)cap, attn::kSeg);
    H3B_REQUIRE(length == 0 || (kq && vq && ks && vs && aligned(kq, 16) && aligned(vq, 16)),
                "h3b_kv8_attn: cache pointers NULL or not 16-byte aligned");
    H3B_REQUIRE(H > 0 && H <= 65535, "h3b_kv8_attn: heads=%lld out of range", (long long)H);
    attn::Args a{};
    a.q = static_cast<const uint16_t*>(q);
    a.q_ld = q_ld, a.q_hs = q_hs;
    a.o = static_cast<uint16_t*>(o);
    a.o_ld = o_ld, a.o_hs = o_hs;
    a.Sq = Sq, a.keys = length, a.H = (int)H, a.scale = scale;
    a.codes[0] = kq, a.codes[1] = vq, a.scales[0] = ks, a.scales[1] = vs, a.cap = cap;
    return attn::launch<true>("h3b_kv8_attn", a, D, static_cast<cudaStream_t>(stream));
}

extern "C" int h3b_block_sparse_attn(const void* q, int64_t q_ld, int64_t q_hs, int64_t Sq, int64_t H, int64_t D,
                                     const void* k, int64_t k_ld, int64_t k_hs, const void* v, int64_t v_ld,
                                     int64_t v_hs, int64_t Sk, const int32_t* blocks, int64_t topk, float scale,
                                     void* o, int64_t o_ld, int64_t o_hs, void* stream) {
    H3B_REQUIRE(topk >= 0 && topk < (1ll << 31) && H > 0 && H <= 65535, "h3b_block_sparse_attn: topk=%lld heads=%lld out of range",
                (long long)topk, (long long)H);
    H3B_REQUIRE(topk == 0 || (blocks && aligned(blocks, 4)), "h3b_block_sparse_attn: blocks NULL");
    H3B_REQUIRE(Sk == 0 || (k && v && aligned(k, 16) && aligned(v, 16)),
                "h3b_block_sparse_attn: k / v NULL or not 16-byte aligned");
    H3B_REQUIRE(k_ld % 8 == 0 && k_hs % 8 == 0 && v_ld % 8 == 0 && v_hs % 8 == 0,
                "h3b_block_sparse_attn: strides must be multiples of 8 elements");
    attn::Args a{};
    a.q = static_cast<const uint16_t*>(q);
    a.q_ld = q_ld, a.q_hs = q_hs;
    a.o = static_cast<uint16_t*>(o);
    a.o_ld = o_ld, a.o_hs = o_hs;
    a.Sq = Sq, a.keys = Sk, a.H = (int)H, a.scale = scale;
    a.kv[0] = static_cast<const uint16_t*>(k), a.kv[1] = static_cast<const uint16_t*>(v);
    a.kv_ld[0] = k_ld, a.kv_hs[0] = k_hs, a.kv_ld[1] = v_ld, a.kv_hs[1] = v_hs;
    a.blocks = blocks, a.topk = (int)topk, a.nq = (Sq + attn::kQRows - 1) / attn::kQRows;
    return attn::launch<false>("h3b_block_sparse_attn", a, D, static_cast<cudaStream_t>(stream));
}
