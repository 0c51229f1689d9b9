// Attention over a key/value cache held in 8 bits, and over selected blocks of
// bf16 keys:  o = softmax(scale * q k^T) v, one pass over the keys with the
// running maximum and sum of the softmax.
#include "ptx.cuh"

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
    int h0;  // first head of the launch
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
    int64_t nq;  // query tiles of 128 rows
    // parts of a split: O [parts, H, Sq, D], (reference maximum, sum) [parts, H, Sq, 2], H of the launch
    float* part_o;
    float* part_ml;
    int* status;
};

// ---------------------------------------------------------------------------
// Tile kernel: 128 query rows of one head per CTA, 128 keys per step.

constexpr int kTileKeys = 128;  // keys per step: two segments
constexpr int kTmemCols = 256;  // S / P: columns 0-127, O: columns 128 ..
constexpr uint64_t kWaitNs = 1000ull * 1000 * 1000;
constexpr float kLog2e = 1.4426950408889634f;
// A row's reference maximum moves when a score exceeds it by 2^8: until then p
// stays below 2^8, far from any limit of fp32 or bf16 (whose relative
// precision does not depend on it), and O is not rescaled.
constexpr float kSlack = 8.0f;

template <int D>
struct Smem {
    static constexpr int kHalves = D / 64;                 // 128-byte column halves of a row
    static constexpr int kTile = kHalves * 128 * 128;      // 128 rows x D bf16
    static constexpr int kQ = 0, kK = kTile, kV = 2 * kTile, kBars = 3 * kTile;
    // at most two CTAs fit beside one another on an SM, as their TMEM does
    static constexpr int kBytes = (3 * kTile + 256 > 80 * 1024) ? 3 * kTile + 256 : 80 * 1024;
};

// kind::f16 instruction descriptor: D fp32 (bits 4-5 = 1), A and B bf16 (7-9 = 1,
// 10-12 = 1), bit 13 negates A, bit 16 = B is MN-major, N >> 3 at 17-22, M >> 4 at 24-28.
constexpr uint32_t idesc(int n, bool b_mn_major) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn_major ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) |
           (8u << 24);
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"((uint32_t)acc)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(id), "r"((uint32_t)acc)
        : "memory");
}
// MN-major operand with 128-byte swizzle: rows are keys (the contraction), 64
// channels each; the next 64 channels lie a half tile (16 KB) on (leading byte
// offset), the next 8 keys 1024 bytes on (stride byte offset).
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(16384 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, const void* src, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map),
                 "r"(smem_u32(src)), "r"(c0), "r"(c1), "r"(c2)
                 : "memory");
}

#define H3B_R16(r, o) "+r"(r[o + 0]), "+r"(r[o + 1]), "+r"(r[o + 2]), "+r"(r[o + 3]), "+r"(r[o + 4]), "+r"(r[o + 5]), \
    "+r"(r[o + 6]), "+r"(r[o + 7]), "+r"(r[o + 8]), "+r"(r[o + 9]), "+r"(r[o + 10]), "+r"(r[o + 11]),                  \
    "+r"(r[o + 12]), "+r"(r[o + 13]), "+r"(r[o + 14]), "+r"(r[o + 15])

// tcgen05.ld of 32 columns without waiting; tmem_ready makes the registers usable.
__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
// Waits for every load so far; naming the registers keeps their uses behind the wait.
__device__ __forceinline__ void tmem_ready(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : H3B_R16(r, 0), H3B_R16(r, 16)::"memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
        "add.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
        "mul.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// Two int8 codes (bytes `sel` picks, zero-extended to 16 bits) -> bf16x2, exactly:
// in [128, 256) a bf16 steps by 1, so 0x4300 | low 7 bits is 128 + them, and
// 0x4300 | sign bit is 128, or 256 for a negative code.
__device__ __forceinline__ uint32_t codes_to_bf16x2(uint32_t x, uint32_t sel) {
    const uint32_t t = __byte_perm(x, 0, sel);
    const uint32_t a = (t & 0x007F007Fu) | 0x43004300u, b = (t & 0x00800080u) | 0x43004300u;
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                     *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&d);
}

// Where the keys and values of a step come from.
enum Source {
    kBlocks,  // selected blocks of bf16 tensors, by TMA
    kWide,    // the cache's codes widened to bf16 beforehand, by TMA
    kCodes,   // the cache's codes, widened by four warps of the CTA
};

// Warps 0-3: softmax, one row a thread; warp 4: the MMAs; after them the
// operand warps, one that issues TMA loads or four that widen codes.
template <Source SRC>
constexpr int tile_threads() {
    return SRC == kCodes ? 288 : 192;
}

// One step's segments: 64 keys each, `n` of them valid, starting at token `at`.
struct Seg {
    int64_t at;
    int n;
};

template <Source SRC>
__device__ __forceinline__ Seg segment(const Args& a, const int32_t* list, int64_t index, int64_t count) {
    if (index >= count) return Seg{a.keys, 0};
    int64_t b = index;
    if constexpr (SRC == kBlocks) {
        b = __ldg(list + index);
        if (b < 0 || b * kSeg >= a.keys) return Seg{a.keys, 0};
    }
    return Seg{b * kSeg, (int)min((int64_t)kSeg, a.keys - b * kSeg)};
}

struct Row {
    float m, l;  // reference maximum (in powers of two) and sum of 2^(x - m)
};

// One step of a row: S (128 columns at tS) -> P (bf16, 64 columns at tS), with
// the running maximum and sum.  n, sk, sv: per segment of 64 keys its valid
// keys, the factor of its scores (softmax scale, log2 e and, for codes, the
// block's scale) and of its values.  TAIL: some keys are not valid.
template <int D, Source SRC, bool TAIL>
__device__ __forceinline__ void softmax_step(Row& st, uint32_t tS, uint32_t tO, bool later, const int (&n)[2],
                                             const float (&sk)[2], const float (&sv)[2]) {
    // with four widening warps in the CTA a thread has too few registers to
    // hold the 128 scores from the maximum to the exponential: they are read twice
    constexpr bool kHold = SRC != kCodes;
    uint32_t r[4][32];
    float mx[2][4];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int c = 0; c < 4; ++c) mx[s][c] = -INFINITY;
    if constexpr (kHold) {
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32_async(tS + c * 32, r[c]);
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ready(r[c]);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        if constexpr (!kHold) {
            tmem_ld32_async(tS + c * 32, r[0]);
            tmem_ready(r[0]);
        }
        const uint32_t(&x)[32] = r[kHold ? c : 0];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
            if (TAIL && (c & 1) * 32 + e >= n[c / 2]) continue;
            mx[c / 2][e & 3] = fmaxf(mx[c / 2][e & 3], __uint_as_float(x[e]));
        }
    }
    float top = -INFINITY;  // the step's largest score
#pragma unroll
    for (int s = 0; s < 2; ++s)
        if (!TAIL || n[s] > 0)
            top = fmaxf(top, fmaxf(fmaxf(mx[s][0], mx[s][1]), fmaxf(mx[s][2], mx[s][3])) * sk[s]);
    const bool moves = top > st.m + kSlack || (st.m == -INFINITY && top > st.m);
    if (__any_sync(0xFFFFFFFFu, moves)) {
        // (this step's S has been waited for, and with it every product before: O stands still)
        const float keep = moves ? ex2(st.m - top) : 1.0f;
        if (moves) st.m = top;
        st.l *= keep;
        if (later) {
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
                uint32_t o[16];
                tmem_ld16(tO + c * 16, o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                tmem_st16(tO + c * 16, o);
            }
        }
    }
    const float ref = st.m == -INFINITY ? 0.0f : st.m;
    float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        if constexpr (!kHold) {
            tmem_ld32_async(tS + c * 32, r[0]);
            tmem_ready(r[0]);
        }
        const uint32_t(&y)[32] = r[kHold ? c : 0];
        const float k = sk[c / 2], v = sv[c / 2];
        uint32_t p[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            float2 x = fma2(make_float2(__uint_as_float(y[2 * e]), __uint_as_float(y[2 * e + 1])), make_float2(k, k),
                            make_float2(-ref, -ref));
            if constexpr (TAIL) {  // behind the product: a scale of zero must not bring a masked key back as NaN
                if ((c & 1) * 32 + 2 * e >= n[c / 2]) x.x = -INFINITY;
                if ((c & 1) * 32 + 2 * e + 1 >= n[c / 2]) x.y = -INFINITY;
            }
            x.x = ex2(x.x);
            x.y = ex2(x.y);
            sum[e & 1] = add2(sum[e & 1], x);
            // p is rounded to bf16 for the second product (its sum is not): a relative 2^-8 at most a key
            if constexpr (SRC != kBlocks) x = mul2(x, make_float2(v, v));
            p[e] = pack_bf16x2(x.x, x.y);
        }
        tmem_st16(tS + c * 16, p);
    }
    sum[0] = add2(sum[0], sum[1]);
    st.l += sum[0].x + sum[0].y;
}

template <int D, Source SRC>
__global__ void __launch_bounds__(tile_threads<SRC>(), 2)
    tile_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmO, Args a) {
    using L = Smem<D>;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* sQ = smem + L::kQ;
    uint8_t* sK = smem + L::kK;
    uint8_t* sV = smem + L::kV;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBars);
    uint64_t *q_full = bars, *k_full = bars + 1, *k_empty = bars + 2, *v_full = bars + 3, *v_empty = bars + 4,
             *s_full = bars + 5, *p_full = bars + 6, *o_full = bars + 7;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 8);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // query tiles first: CTAs that run together share a head's keys in L2
    const int64_t qt = blockIdx.x % (unsigned)a.nq;
    const int hl = (int)(blockIdx.x / (unsigned)a.nq);  // head within the launch
    const int h = a.h0 + hl;
    const int32_t* list = SRC == kBlocks ? a.blocks + ((int64_t)h * a.nq + qt) * a.topk : nullptr;
    const int64_t segs = SRC == kBlocks ? a.topk : (a.keys + kSeg - 1) / kSeg;
    const int64_t steps_all = (segs + 1) / 2;
    const int64_t step0 = steps_all * blockIdx.y / gridDim.y;
    const int steps = (int)(steps_all * (blockIdx.y + 1) / gridDim.y - step0);

    // the swizzled tiles need the 1024-byte alignment that this declaration asks for
    if (smem_u32(smem) & 1023u) {
        if (threadIdx.x == 0) report(a.status, H3B_STATUS_MBAR_TIMEOUT);
        return;
    }
    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        mbar_init(k_full, SRC == kCodes ? 4 : 1);
        mbar_init(v_full, SRC == kCodes ? 4 : 1);
        mbar_init(k_empty, 1);
        mbar_init(v_empty, 1);
        mbar_init(s_full, 1);
        mbar_init(p_full, 4);
        mbar_init(o_full, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 4) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint32_t tS = tmem, tO = tmem + 128u;

    if (warp == 4) {
        // ---------------- MMA issuer (and the load of Q)
        if (lane == 0 && steps > 0) {
            mbar_expect_tx(q_full, L::kTile);
#pragma unroll
            for (int c = 0; c < L::kHalves; ++c)
                tma_load_3d(sQ + c * 16384, &tmQ, q_full, c * 64, h, (int)(qt * kQRows));
            const uint32_t id_s = idesc(kTileKeys, false) | (a.scale < 0.0f ? 1u << 13 : 0u);
            const uint32_t id_o = idesc(D, true);
            const uint32_t q0 = smem_u32(sQ), k0 = smem_u32(sK), v0 = smem_u32(sV);
            bool ok = mbar_wait(q_full, 0, abort_flag, a.status, kWaitNs);
            for (int i = 0; ok && i <= steps; ++i) {
                if (i > 0) {
                    // O += P V of the step before
                    const uint32_t ph = (uint32_t)(i - 1) & 1u;
                    ok = mbar_wait(v_full, ph, abort_flag, a.status, kWaitNs) &&
                         mbar_wait(p_full, ph, abort_flag, a.status, kWaitNs);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int k = 0; k < kTileKeys / 16; ++k)
                        mma_ts(tO, tS + 8 * k, smem_desc_mn(v0 + k * 2048), id_o, (i - 1) | k);
                    umma_commit(v_empty);
                }
                if (i < steps) {
                    // S = Q K^T: it takes the place of P, which the product before has read (MMAs run in order)
                    ok = mbar_wait(k_full, (uint32_t)i & 1u, abort_flag, a.status, kWaitNs);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int k = 0; k < D / 16; ++k)
                        mma_ss(tS, smem_desc(q0 + (k / 4) * 16384 + (k % 4) * 32),
                               smem_desc(k0 + (k / 4) * 16384 + (k % 4) * 32), id_s, k);
                    umma_commit(k_empty);
                    umma_commit(s_full);
                }
            }
            // on every way out: no MMA of this thread stays in flight
            umma_commit(o_full);
            if (!ok) {
                volatile int no_abort = 0;
                mbar_wait(o_full, 0, &no_abort, nullptr, 100ull * 1000 * 1000);
            }
        }
        __syncwarp();
    } else if (warp > 4) {
        if constexpr (SRC == kCodes) {
            // ---------------- codes -> bf16 tiles
            constexpr int kLanes = D / 16;          // threads along a token's channels, 16 codes each
            constexpr int kRows = 128 / kLanes;     // tokens per pass
            constexpr int kPasses = kTileKeys / kRows;
            const int t = threadIdx.x - 160;
            const int col = t % kLanes, row = t / kLanes;
            const int8_t* src[2];
#pragma unroll
            for (int w = 0; w < 2; ++w) src[w] = a.codes[w] + (int64_t)h * a.cap * D + col * 16;
            uint4 held[2][kPasses];
            auto fetch = [&](int w, int i) {
                const int64_t tok = (step0 + i) * kTileKeys + row;
#pragma unroll
                for (int p = 0; p < kPasses; ++p) {
                    held[w][p] = make_uint4(0, 0, 0, 0);
                    if (tok + p * kRows < a.keys)
                        held[w][p] = __ldg(reinterpret_cast<const uint4*>(src[w] + (tok + p * kRows) * D));
                }
            };
            auto store = [&](int w, uint8_t* tile) {
                // 16 codes become two 16-byte pieces of the row's 128-byte half; the lanes of the upper half
                // store them in the other order, so that eight lanes meet eight bank groups
                uint8_t* half = tile + (col / 4) * 16384;
                const int first = (col >> 2) & 1;
#pragma unroll
                for (int p = 0; p < kPasses; ++p) {
                    const int r = row + p * kRows;
                    const uint4 x = held[w][p];
                    const uint4 lo = make_uint4(codes_to_bf16x2(x.x, 0x4140), codes_to_bf16x2(x.x, 0x4342),
                                                codes_to_bf16x2(x.y, 0x4140), codes_to_bf16x2(x.y, 0x4342));
                    const uint4 hi = make_uint4(codes_to_bf16x2(x.z, 0x4140), codes_to_bf16x2(x.z, 0x4342),
                                                codes_to_bf16x2(x.w, 0x4140), codes_to_bf16x2(x.w, 0x4342));
                    const int c0 = (col % 4) * 2 + first;
                    *reinterpret_cast<uint4*>(half + r * 128 + ((c0 ^ (r & 7)) << 4)) = first ? hi : lo;
                    *reinterpret_cast<uint4*>(half + r * 128 + (((c0 ^ 1) ^ (r & 7)) << 4)) = first ? lo : hi;
                }
            };
            if (steps > 0) {
                fetch(0, 0);
                fetch(1, 0);
            }
            for (int i = 0; i < steps; ++i) {
                const uint32_t ph = ((uint32_t)i & 1u) ^ 1u;
                if (!mbar_wait(k_empty, ph, abort_flag, a.status, kWaitNs)) break;
                store(0, sK);
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(k_full);
                if (i + 1 < steps) fetch(0, i + 1);
                if (!mbar_wait(v_empty, ph, abort_flag, a.status, kWaitNs)) break;
                store(1, sV);
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(v_full);
                if (i + 1 < steps) fetch(1, i + 1);
            }
        } else if (lane == 0) {
            // ---------------- TMA loads; what is not there (a gap in the list, keys behind the last) lies
            // outside the tensor and arrives as zeros
            bool ok = true;
            int k_armed = 0, v_armed = 0;
            for (int i = 0; ok && i < steps; ++i) {
                const uint32_t ph = ((uint32_t)i & 1u) ^ 1u;
                int at[2];
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const int64_t index = 2 * (step0 + i) + s;
                    at[s] = (int)segment<SRC>(a, list, index, segs).at;
                    if (SRC == kBlocks && index < segs) {
                        const int64_t b = __ldg(list + index);
                        if (b < -1 || b * kSeg >= a.keys) report(a.status, H3B_STATUS_BAD_INDEX);
                    }
                }
#pragma unroll
                for (int w = 0; w < 2 && ok; ++w) {
                    uint64_t* full = w ? v_full : k_full;
                    if (!mbar_wait(w ? v_empty : k_empty, ph, abort_flag, a.status, kWaitNs)) {
                        ok = false;
                        break;
                    }
                    mbar_expect_tx(full, L::kTile);
#pragma unroll
                    for (int s = 0; s < 2; ++s)
#pragma unroll
                        for (int c = 0; c < L::kHalves; ++c)
                            tma_load_3d((w ? sV : sK) + c * 16384 + s * 8192, w ? &tmV : &tmK, full, c * 64,
                                        SRC == kBlocks ? h : hl, at[s]);
                    ++(w ? v_armed : k_armed);
                }
            }
            if (!ok) {
                // let the loads in flight land before the CTA exits
                volatile int no_abort = 0;
                if (k_armed) mbar_wait(k_full, (uint32_t)(k_armed - 1) & 1u, &no_abort, nullptr, 100ull * 1000 * 1000);
                if (v_armed) mbar_wait(v_full, (uint32_t)(v_armed - 1) & 1u, &no_abort, nullptr, 100ull * 1000 * 1000);
            }
        }
        __syncwarp();
    } else {
        // ---------------- softmax, one query row a thread
        const uint32_t at = (uint32_t)(warp * 32) << 16;
        const int64_t row = qt * kQRows + threadIdx.x;
        const float scale2 = fabsf(a.scale) * kLog2e;
        Row st{-INFINITY, 0.0f};
        bool ok = true;
        for (int i = 0; i < steps; ++i) {
            int n[2];
            float sk[2], sv[2];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const Seg g = segment<SRC>(a, list, 2 * (step0 + i) + s, segs);
                n[s] = g.n;
                sk[s] = scale2;
                sv[s] = 1.0f;
                if (SRC != kBlocks && g.n > 0) {
                    sk[s] = scale2 * __ldg(a.scales[0] + (int64_t)h * (a.cap / kSeg) + g.at / kSeg);
                    sv[s] = __ldg(a.scales[1] + (int64_t)h * (a.cap / kSeg) + g.at / kSeg);
                }
            }
            if (!(ok = mbar_wait(s_full, (uint32_t)i & 1u, abort_flag, a.status, kWaitNs))) break;
            tc_fence_after();
            if (n[0] + n[1] == kTileKeys)
                softmax_step<D, SRC, false>(st, tS + at, tO + at, i > 0, n, sk, sv);
            else
                softmax_step<D, SRC, true>(st, tS + at, tO + at, i > 0, n, sk, sv);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full);
        }
        const float m = st.m, l = st.l;
        if (ok && steps > 0) ok = mbar_wait(o_full, 0, abort_flag, a.status, kWaitNs);
        tc_fence_after();
        if (ok && gridDim.y > 1) {
            // a part of the keys: O, its reference maximum and sum go to the join
            const int64_t part = (int64_t)blockIdx.y * gridDim.x / a.nq * a.Sq + (int64_t)hl * a.Sq + row;
            if (row < a.Sq) {
                a.part_ml[2 * part] = m;
                a.part_ml[2 * part + 1] = l;
            }
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                uint32_t r[32];
                if (steps > 0) {
                    tmem_ld32_async(tO + at + c * 32, r);
                    tmem_ready(r);
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) r[e] = 0;
                }
                if (row < a.Sq) {
                    uint4* dst = reinterpret_cast<uint4*>(a.part_o + part * D + c * 32);
#pragma unroll
                    for (int e = 0; e < 8; ++e) dst[e] = make_uint4(r[4 * e], r[4 * e + 1], r[4 * e + 2], r[4 * e + 3]);
                }
            }
        } else if (ok) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            // through Q's place in shared memory (every MMA is done) into whole rows of o
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                uint32_t r[32];
                if (steps > 0) {
                    tmem_ld32_async(tO + at + c * 32, r);
                    tmem_ready(r);
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) r[e] = 0;
                }
                uint8_t* half = sQ + (c / 2) * 16384 + threadIdx.x * 128;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t o[4];
#pragma unroll
                    for (int f = 0; f < 4; ++f)
                        o[f] = pack_bf16x2(__uint_as_float(r[8 * e + 2 * f]) * inv, __uint_as_float(r[8 * e + 2 * f + 1]) * inv);
                    *reinterpret_cast<uint4*>(half + ((((c & 1) * 4 + e) ^ (threadIdx.x & 7)) << 4)) =
                        make_uint4(o[0], o[1], o[2], o[3]);
                }
            }
            fence_async_smem();
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (gridDim.y == 1 && !*abort_flag && threadIdx.x == 0) {
#pragma unroll
            for (int c = 0; c < L::kHalves; ++c) tma_store_3d(&tmO, sQ + c * 16384, c * 64, h, (int)(qt * kQRows));
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        }
        __syncwarp();
    }

    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 4)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

// Join of the parts of a split: o = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s.  One warp a row.
template <int D>
__global__ void __launch_bounds__(128) join_kernel(Args a, int heads, int parts) {
    const int lane = threadIdx.x & 31;
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int64_t step = a.Sq * heads;
    if (id >= step) return;
    const int h = a.h0 + (int)(id / a.Sq);
    const int64_t row = id % a.Sq;
    float m = -INFINITY;
    for (int s = lane; s < parts; s += 32) m = fmaxf(m, a.part_ml[2 * (s * step + id)]);
#pragma unroll
    for (int off = 16; off; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, off));
    const float ref = m == -INFINITY ? 0.0f : m;
    float l = 0.0f, o[D / 32] = {};
    for (int s = 0; s < parts; ++s) {
        const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * (s * step + id));
        const float w = ex2(ml.x - ref);
        l += w * ml.y;
#pragma unroll
        for (int e = 0; e < D / 32; ++e) o[e] += w * a.part_o[(s * step + id) * D + lane * (D / 32) + e];
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint16_t* dst = a.o + row * a.o_ld + h * a.o_hs + lane * (D / 32);
#pragma unroll
    for (int e = 0; e < D / 32; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = pack_bf16x2(o[e] * inv, o[e + 1] * inv);
}

// Codes of some heads (each `per` pieces of 16 from `stride` pieces apart) -> bf16, K or V by blockIdx.y.
__global__ void __launch_bounds__(256) widen_kernel(const int8_t* __restrict__ kq, const int8_t* __restrict__ vq,
                                                    int64_t stride, int64_t per, int64_t pieces,
                                                    uint16_t* __restrict__ k, uint16_t* __restrict__ v) {
    const uint4* src = reinterpret_cast<const uint4*>(blockIdx.y ? vq : kq);
    uint4* dst = reinterpret_cast<uint4*>(blockIdx.y ? v : k);
    uint4 x[4];
    const int64_t first = (int64_t)blockIdx.x * 1024 + threadIdx.x;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const int64_t i = first + p * 256;
        if (i < pieces) x[p] = __ldg(src + i / per * stride + i % per);
    }
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const int64_t i = first + p * 256;
        if (i >= pieces) break;
        dst[2 * i] = make_uint4(codes_to_bf16x2(x[p].x, 0x4140), codes_to_bf16x2(x[p].x, 0x4342),
                                codes_to_bf16x2(x[p].y, 0x4140), codes_to_bf16x2(x[p].y, 0x4342));
        dst[2 * i + 1] = make_uint4(codes_to_bf16x2(x[p].z, 0x4140), codes_to_bf16x2(x[p].z, 0x4342),
                                    codes_to_bf16x2(x[p].w, 0x4140), codes_to_bf16x2(x[p].w, 0x4342));
    }
}

// [tokens, heads, D] bf16 as boxes of `rows` tokens x 64 channels of a head.
static int make_map(CUtensorMap* map, const void* p, int64_t n, int H, int64_t D, int64_t ld, int64_t hs, int rows) {
    PFN_encodeTiled enc = encode_fn();
    if (!enc) return set_error(H3B_ERR_CUDA, "cuTensorMapEncodeTiled unavailable (driver too old?)");
    cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)H, (cuuint64_t)n};
    cuuint64_t strides[2] = {(cuuint64_t)hs * 2, (cuuint64_t)ld * 2};
    cuuint32_t box[3] = {64, 1, (cuuint32_t)rows};
    cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(p), dims, strides, box, estr,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(H3B_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return H3B_OK;
}

static int sm_count() {
    static int cached = 0;
    if (!cached) {
        int dev = 0, n = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
            return 148;
        cached = n;
    }
    return cached;
}

// Parts that the keys of every row tile are split into.  All CTAs take about as
// long, so the time is the number of rounds of two CTAs an SM times a part's
// steps plus what a CTA spends besides (about two steps); a join costs about
// two more.
static int64_t parts_of(int64_t tiles, int64_t steps) {
    const int64_t room = 2 * sm_count();
    int64_t best = 1, best_cost = 0;
    for (int64_t n = 1; n <= 64 && (n == 1 || n * 2 <= steps); ++n) {
        const int64_t cost = cdiv(tiles * n, room) * (cdiv(steps, n) + 2) + (n > 1 ? 2 : 0);
        if (n == 1 || cost < best_cost) best = n, best_cost = cost;
    }
    return best;
}

struct Plan {
    bool wide;          // the cache's codes are widened beforehand
    int64_t heads;      // heads a launch (and of the widened copy)
    int64_t parts;      // of the keys
    int64_t join_at, bytes;  // in the workspace
};

// From this many row tiles on a head's codes are widened once instead of by every CTA.
constexpr int64_t kWideTiles = 4;
constexpr int64_t kWideBytes = 256ll << 20;  // of widened heads at a time (one head at least)

static Plan plan(bool cache, int64_t Sq, int64_t H, int64_t D, int64_t segs) {
    Plan p{};
    const int64_t nq = cdiv(Sq, kQRows);
    p.wide = cache && nq >= kWideTiles && segs > 0;
    const int64_t head = 2 * segs * kSeg * D * 2;
    p.heads = H;
    if (p.wide && H * head > kWideBytes) p.heads = kWideBytes / head > 0 ? kWideBytes / head : 1;
    p.parts = parts_of(nq * p.heads, cdiv(segs, 2));
    p.join_at = p.wide ? p.heads * head : 0;
    p.bytes = p.join_at + (p.parts > 1 ? p.parts * p.heads * Sq * (D + 2) * 4 : 0);
    return p;
}

template <int D, Source SRC>
static int launch_tiles(Args a, int64_t heads, int64_t parts, const uint16_t* const (&kv)[2], const int64_t (&ld)[2],
                        const int64_t (&hs)[2], cudaStream_t s) {
    CUtensorMap q{}, k{}, v{}, o{};
    if (int rc = make_map(&q, a.q, a.Sq, a.H, D, a.q_ld, a.q_hs, kQRows)) return rc;
    if (int rc = make_map(&o, a.o, a.Sq, a.H, D, a.o_ld, a.o_hs, kQRows)) return rc;
    if (SRC != kCodes && a.keys > 0) {
        const int n = SRC == kBlocks ? a.H : (int)heads;
        if (int rc = make_map(&k, kv[0], a.keys, n, D, ld[0], hs[0], kSeg)) return rc;
        if (int rc = make_map(&v, kv[1], a.keys, n, D, ld[1], hs[1], kSeg)) return rc;
    }
    H3B_CUDA_TRY(cudaFuncSetAttribute(tile_kernel<D, SRC>, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<D>::kBytes));
    const dim3 grid((unsigned)(a.nq * heads), (unsigned)parts);
    tile_kernel<D, SRC><<<grid, tile_threads<SRC>(), Smem<D>::kBytes, s>>>(q, k, v, o, a);
    if (parts > 1) join_kernel<D><<<(unsigned)cdiv(a.Sq * heads, 4), 128, 0, s>>>(a, (int)heads, (int)parts);
    H3B_CUDA_TRY(cudaGetLastError());
    return H3B_OK;
}

template <int D>
static int launch_all(Args& a, bool cache, const Plan& p, int64_t segs, char* ws, cudaStream_t s) {
    a.part_o = reinterpret_cast<float*>(ws + p.join_at);
    a.part_ml = a.part_o + (p.parts > 1 ? p.parts * p.heads * a.Sq * D : 0);
    if (!cache) return launch_tiles<D, kBlocks>(a, a.H, p.parts, a.kv, a.kv_ld, a.kv_hs, s);
    if (!p.wide) return launch_tiles<D, kCodes>(a, a.H, p.parts, a.kv, a.kv_ld, a.kv_hs, s);
    const int64_t rows = segs * kSeg;
    uint16_t* const k = reinterpret_cast<uint16_t*>(ws);
    for (int64_t h = 0; h < a.H; h += p.heads) {
        const int64_t n = a.H - h < p.heads ? a.H - h : p.heads;
        uint16_t* const v = k + n * rows * D;
        const int64_t pieces = n * rows * D / 16;
        widen_kernel<<<dim3((unsigned)cdiv(pieces, 4 * 256), 2), 256, 0, s>>>(
            a.codes[0] + h * a.cap * D, a.codes[1] + h * a.cap * D, a.cap * D / 16, rows * D / 16, pieces, k, v);
        a.h0 = (int)h;
        const int64_t ld[2] = {D, D}, hs[2] = {rows * D, rows * D};
        const uint16_t* const kv[2] = {k, v};
        if (int rc = launch_tiles<D, kWide>(a, n, p.parts, kv, ld, hs, s)) return rc;
    }
    return H3B_OK;
}

static int launch(const char* who, bool cache, Args& a, int64_t D, int64_t segs, void* ws, int64_t ws_bytes,
                  cudaStream_t s) {
    H3B_REQUIRE(D == 64 || D == 128, "%s: head_dim=%lld must be 64 or 128", who, (long long)D);
    H3B_REQUIRE(a.Sq >= 0 && a.keys >= 0 && a.H > 0 && a.H <= 65535 && a.Sq < (1ll << 31) - 128 &&
                    a.keys < (1ll << 31) - 128,
                "%s: shape out of range (rows=%lld keys=%lld heads=%d)", who, (long long)a.Sq, (long long)a.keys, a.H);
    if (a.Sq == 0) return H3B_OK;
    H3B_REQUIRE(a.q && a.o && aligned(a.q, 16) && aligned(a.o, 16), "%s: q / o NULL or not 16-byte aligned", who);
    H3B_REQUIRE(a.q_ld > 0 && a.q_hs > 0 && a.o_ld > 0 && a.o_hs > 0 && a.q_ld % 8 == 0 && a.q_hs % 8 == 0 &&
                    a.o_ld % 8 == 0 && a.o_hs % 8 == 0,
                "%s: strides must be positive multiples of 8 elements", who);
    a.nq = cdiv(a.Sq, kQRows);
    H3B_REQUIRE(a.nq * a.H < (1ll << 31) && a.Sq * a.H < (1ll << 33), "%s: too many row tiles", who);
    const Plan p = plan(cache, a.Sq, a.H, D, segs);
    H3B_REQUIRE(p.bytes == 0 || (ws && aligned(ws, 256) && ws_bytes >= p.bytes),
                "%s: workspace of %lld bytes (256-byte aligned), %lld needed", who, (long long)ws_bytes, (long long)p.bytes);
    DeviceStatus ds;
    if (int rc = device_status(&ds)) return rc;
    a.status = ds.word;
    return D == 128 ? launch_all<128>(a, cache, p, segs, static_cast<char*>(ws), s)
                    : launch_all<64>(a, cache, p, segs, static_cast<char*>(ws), s);
}

}  // namespace attn
}  // namespace h3b

using namespace h3b;

extern "C" int64_t h3b_attn_workspace(int cache, int64_t Sq, int64_t H, int64_t D, int64_t segments) {
    if (Sq <= 0 || H <= 0 || segments <= 0 || (D != 64 && D != 128)) return 0;
    return attn::plan(cache != 0, Sq, H, D, segments).bytes;
}

extern "C" int h3b_kv8_attn(const void* q, int64_t q_ld, int64_t q_hs, int64_t Sq, int64_t H, int64_t D,
                            const int8_t* kq, const int8_t* vq, const float* ks, const float* vs, int64_t cap,
                            int64_t length, float scale, void* o, int64_t o_ld, int64_t o_hs, void* workspace,
                            int64_t workspace_bytes, void* stream) {
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
    return attn::launch("h3b_kv8_attn", true, a, D, cdiv(length, attn::kSeg), workspace, workspace_bytes,
                              static_cast<cudaStream_t>(stream));
}

extern "C" int h3b_block_sparse_attn(const void* q, int64_t q_ld, int64_t q_hs, int64_t Sq, int64_t H, int64_t D,
                                     const void* k, int64_t k_ld, int64_t k_hs, const void* v, int64_t v_ld,
                                     int64_t v_hs, int64_t Sk, const int32_t* blocks, int64_t topk, float scale,
                                     void* o, int64_t o_ld, int64_t o_hs, void* workspace, int64_t workspace_bytes,
                                     void* stream) {
    H3B_REQUIRE(topk >= 0 && topk < (1ll << 31) && H > 0 && H <= 65535, "h3b_block_sparse_attn: topk=%lld heads=%lld out of range",
                (long long)topk, (long long)H);
    H3B_REQUIRE(topk == 0 || (blocks && aligned(blocks, 4)), "h3b_block_sparse_attn: blocks NULL");
    H3B_REQUIRE(Sk == 0 || (k && v && aligned(k, 16) && aligned(v, 16)),
                "h3b_block_sparse_attn: k / v NULL or not 16-byte aligned");
    H3B_REQUIRE(k_ld > 0 && k_hs > 0 && v_ld > 0 && v_hs > 0 && k_ld % 8 == 0 && k_hs % 8 == 0 && v_ld % 8 == 0 &&
                    v_hs % 8 == 0,
                "h3b_block_sparse_attn: strides must be positive multiples of 8 elements");
    attn::Args a{};
    a.q = static_cast<const uint16_t*>(q);
    a.q_ld = q_ld, a.q_hs = q_hs;
    a.o = static_cast<uint16_t*>(o);
    a.o_ld = o_ld, a.o_hs = o_hs;
    a.Sq = Sq, a.keys = Sk, a.H = (int)H, a.scale = scale;
    a.kv[0] = static_cast<const uint16_t*>(k), a.kv[1] = static_cast<const uint16_t*>(v);
    a.kv_ld[0] = k_ld, a.kv_hs[0] = k_hs, a.kv_ld[1] = v_ld, a.kv_hs[1] = v_hs;
    a.blocks = blocks, a.topk = (int)topk;
    return attn::launch("h3b_block_sparse_attn", false, a, D, topk, workspace, workspace_bytes,
                               static_cast<cudaStream_t>(stream));
}
