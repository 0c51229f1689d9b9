// Block-sparse attention in one call: the means of the query and key blocks, the
// selection and the attention over it, enqueued one behind the other.
#include "common.cuh"

namespace h3b {
int sparse_means(const void* k, int64_t k_ld, int64_t k_hs, int64_t Sk, float* km, const void* q, int64_t q_ld,
                 int64_t q_hs, int64_t Sq, float* qm, int64_t H, int64_t D, cudaStream_t s);
}  // namespace h3b

using namespace h3b;

namespace {

constexpr int64_t kKeys = 64, kQRows = 128;

struct Layout {
    int64_t nq, nk, topk;
    int64_t qm, km, select, attn, bytes;  // offsets in the workspace, and its size
};

int64_t up(int64_t n) { return (n + 255) / 256 * 256; }

Layout layout(int64_t Sq, int64_t Sk, int64_t H, int64_t D, int64_t topk, bool means) {
    Layout l{};
    l.nq = cdiv(Sq, kQRows);
    l.nk = cdiv(Sk, kKeys);
    l.topk = topk < l.nk ? topk : l.nk;
    l.km = up(l.nq * H * D * 4);
    l.select = l.km + (means ? 0 : up(l.nk * H * D * 4));
    // the scores are done with when the attention begins
    l.attn = l.select;
    const int64_t a = l.topk > 0 ? h3b_select_blocks_workspace(l.nq, l.nk, H) : 0, b = h3b_attn_workspace(0, Sq, H, D, l.topk);
    l.bytes = l.select + (a > b ? a : b);
    return l;
}

bool sane(int64_t Sq, int64_t Sk, int64_t H, int64_t D, int64_t topk) {
    return Sq >= 0 && Sk >= 0 && H > 0 && H <= 65535 && (D == 64 || D == 128) && topk >= 0 && Sq < (1ll << 31) - 128 &&
           Sk < (1ll << 31) - 128;
}

}  // namespace

extern "C" int64_t h3b_sparse_attn_workspace(int64_t Sq, int64_t Sk, int64_t H, int64_t D, int64_t topk, int has_means) {
    return sane(Sq, Sk, H, D, topk) ? layout(Sq, Sk, H, D, topk, has_means != 0).bytes : 0;
}

extern "C" int h3b_sparse_attn(const void* q, int64_t q_ld, int64_t q_hs, int64_t Sq, int64_t H, int64_t D, const void* k,
                               int64_t k_ld, int64_t k_hs, const void* v, int64_t v_ld, int64_t v_hs, int64_t Sk,
                               const float* k_means, int64_t topk, float scale, int32_t* blocks, void* o, int64_t o_ld,
                               int64_t o_hs, void* workspace, int64_t workspace_bytes, void* stream) {
    H3B_REQUIRE(sane(Sq, Sk, H, D, topk),
                "h3b_sparse_attn: rows=%lld keys=%lld heads=%lld head_dim=%lld (64 or 128) topk=%lld out of range",
                (long long)Sq, (long long)Sk, (long long)H, (long long)D, (long long)topk);
    const Layout l = layout(Sq, Sk, H, D, topk, k_means != nullptr);
    H3B_REQUIRE(l.bytes == 0 || (workspace && aligned(workspace, 256) && workspace_bytes >= l.bytes),
                "h3b_sparse_attn: workspace of %lld bytes (256-byte aligned), %lld needed", (long long)workspace_bytes,
                (long long)l.bytes);
    // (what the attention would refuse, before the means and the selection are under way)
    H3B_REQUIRE(Sq == 0 || (q && o && aligned(q, 16) && aligned(o, 16)), "h3b_sparse_attn: q / o NULL or not 16-byte aligned");
    H3B_REQUIRE(Sk == 0 || (k && v && aligned(k, 16) && aligned(v, 16)), "h3b_sparse_attn: k / v NULL or not 16-byte aligned");
    H3B_REQUIRE(Sq == 0 || l.topk == 0 || (blocks && aligned(blocks, 4)), "h3b_sparse_attn: blocks NULL");
    for (const int64_t stride : {q_ld, q_hs, k_ld, k_hs, v_ld, v_hs, o_ld, o_hs})
        H3B_REQUIRE(stride > 0 && stride % 8 == 0, "h3b_sparse_attn: strides must be positive multiples of 8 elements");
    char* ws = static_cast<char*>(workspace);
    float *qm = reinterpret_cast<float*>(ws + l.qm), *km = reinterpret_cast<float*>(ws + l.km);
    if (l.topk > 0 && Sq > 0) {
        if (int rc = sparse_means(k, k_ld, k_hs, Sk, k_means ? nullptr : km, q, q_ld, q_hs, Sq, qm, H, D,
                                  static_cast<cudaStream_t>(stream)))
            return rc;
        if (int rc = h3b_select_blocks(qm, k_means ? k_means : km, l.nq, l.nk, H, D, l.topk, blocks, ws + l.select,
                                       workspace_bytes - l.select, stream))
            return rc;
    }
    return h3b_block_sparse_attn(q, q_ld, q_hs, Sq, H, D, k, k_ld, k_hs, v, v_ld, v_hs, Sk, blocks, l.topk, scale, o, o_ld,
                                 o_hs, ws + l.attn, workspace_bytes - l.attn, stream);
}
