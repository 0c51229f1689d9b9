// Attention over a key/value cache held in 8 bits, and over selected blocks of
// bf16 keys:  o = softmax(scale * q k^T) v, one pass over the keys with the
// running maximum and sum of the softmax.
#include <cuda_fp16.h>

#include <type_traits>

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
    int64_t segs;   // segments of 64 keys
    uint32_t items;  // pairs of tiles of the launch
    int heads, parts;  // heads of the launch, parts of the keys
    bool turns;        // the exponentials of a pair's tiles take turns
    // parts of a split: O [parts, H, Sq, D], (reference maximum, sum) [parts, H, Sq, 2], H of the launch
    float* part_o;
    float* part_ml;
    int* status;
};

// ---------------------------------------------------------------------------
// Pair kernel: a persistent CTA per SM works on two tiles of 128 query rows at a
// time, 64 keys a step each.
//
// A step of a tile is a chain: S = Q K^T (tensor cores), softmax of S (its own
// four warps, one row a thread), O += P V (tensor cores).  TMEM holds, per tile,
// O and two S of 64 columns (P takes the place of its S), so that the next
// step's S is there when a softmax ends, and neither the softmax warps nor the
// tensor cores wait for a chain to go round.  (One S of 128 columns a tile, the
// other form that fits in TMEM, left the tensor cores idle more than half of the
// time: the chain of a step took 3700 clocks, of which 1024 are products.)
// What bounds it: shared memory in part (the operands of Q K^T alone take its 128
// bytes a clock for 384 clocks a step and tile, where the products take 256: 1280
// clocks a step of both tiles), the chain of a step and the power cap for the
// rest (1950 measured).  128000 rows of 5 heads over 64 blocks each: 1.28 ms, 1050
// TFLOP/s.

constexpr int kTmemCols = 512;     // S of tile t at 128 t (+ 64 for odd steps), O at 256 + 128 t
constexpr int kPairThreads = 384;  // 2 x 4 softmax warps, an MMA warp and a TMA warp for each tile
constexpr float kLog2e = 1.4426950408889634f;
// A row's reference maximum moves when a score exceeds it by 2^8: until then p
// stays below 2^8, far from any limit of fp32 or bf16 (whose relative
// precision does not depend on it), and O is not rescaled.
constexpr float kSlack = 8.0f;
// The maximum that a part of a split passes on where it has keys whose scores are all
// -infinity; -infinity itself: no keys.  (Rows without a key are zero, rows of such scores NaN.)
constexpr float kLowest = -3.402823466e38f;

template <int D>
struct Smem {
    static constexpr int kHalves = D / 64;             // 128-byte column halves of a row
    static constexpr int kTile = kHalves * 128 * 128;  // 128 rows x D bf16: Q, O
    static constexpr int kSegHalf = kSeg * 128;        // 64 keys of a half
    static constexpr int kSegTile = kHalves * kSegHalf;
    // K and V arrive in groups: the keys of a step with the values of the step two before it
    static constexpr int kGroup = 2 * kSegTile, kGroups = 4;
    static constexpr int kQ = 0, kKV = 2 * kTile, kO = kKV + kGroups * kGroup, kBars = kO + kTile;
    static constexpr int kBytes = kBars + 512;
};

// kind::f16 instruction descriptor: D fp32 (bits 4-5 = 1), A and B bf16 (7-9 = 1,
// 10-12 = 1), bit 13 negates A, bit 16 = B is MN-major, N >> 3 at 17-22, M >> 4 at 24-28.
constexpr uint32_t idesc(int n, bool b_mn_major) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn_major ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) |
           (8u << 24);
}

// Shared-memory descriptors are built inside the MMA's asm from a low word (start
// address >> 4, leading byte offset >> 4 at bit 16), which stepping along the
// operand only adds to, and a constant high word: stride byte offset 1024 (8 rows
// of 128 bytes), version 1, 128-byte swizzle.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
// K-major: rows of 64 channels; the leading byte offset is not used.
__device__ __forceinline__ uint32_t desc_k(const void* p) { return ((smem_u32(p) >> 4) & 0x3FFFu) | (1u << 16); }
// MN-major (V): rows are keys, the contraction, of 64 channels each; the next 64
// channels lie kSeg rows on, the leading byte offset.
__device__ __forceinline__ uint32_t desc_mn(const void* p) {
    return ((smem_u32(p) >> 4) & 0x3FFFu) | (((uint32_t)kSeg * 128u >> 4) << 16);
}

// D (TMEM) [+]= A (shared memory) B^T
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 x, {%1, %5};\n\tmov.b64 y, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(id), "r"(acc), "n"(kDescHi)
        : "memory");
}
// the same with A in TMEM
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 y, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(id), "r"(acc), "n"(kDescHi)
        : "memory");
}

// [tokens, heads, D] bf16 seen as (64 channels, tokens, halves of D, heads): a box
// lands as whole 128-byte rows, the halves of D one behind the other.
__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* map, uint64_t* bar, int token, int head) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %3, %5}], [%2];" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(smem_u32(bar)), "r"(0), "r"(token), "r"(head)
        : "memory");
}
__device__ __forceinline__ void tma_store(const CUtensorMap* map, const void* src, int token, int head) {
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %2, %4}], [%1];" ::"l"(map),
                 "r"(smem_u32(src)), "r"(0), "r"(token), "r"(head)
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

// max of three, NaN if one of them is
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Two int8 codes (in bytes 0 and 2; what is in the others does not matter) ->
// bf16x2, exactly: in [128, 256) a bf16 steps by 1, so 0x4300 | low 7 bits is 128
// + them, and 0x4300 | sign bit is 128, or 256 for a negative code.
__device__ __forceinline__ uint32_t widen2(uint32_t t) {
    const uint32_t a = (t & 0x007F007Fu) | 0x43004300u, b = (t & 0x00800080u) | 0x43004300u;
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                     *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&d);
}
// bytes 0 and 1 (sel 0x4140) or 2 and 3 (0x4342) of a word
__device__ __forceinline__ uint32_t codes_to_bf16x2(uint32_t x, uint32_t sel) { return widen2(__byte_perm(x, 0, sel)); }
// Where a tile's keys and values come from.
enum Source {
    kBlocks,  // selected blocks of bf16 tensors, each tile its own
    kWide,    // the cache's codes widened to bf16 beforehand, the same for both tiles of a pair
};

// One step's segment: 64 keys, `n` of them valid, starting at token `at`.
struct Seg {
    int at, n;
};

struct Row {
    float m, l;  // reference maximum (in powers of two) and sum of 2^(x - m)
};

// Bounded wait for a phase.  False if the wait gave up or another role has.  (A
// barrier is shared memory, which the products' operands keep busy: a look at
// one takes some 250 clocks here, so what can be is asked for together.)
__device__ __forceinline__ bool await(uint64_t* bar, uint32_t phase, volatile int* abort_flag, int* status) {
    uint64_t t0 = 0;
    for (;;) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(phase & 1u)
            : "memory");
        if (ok) return true;
        if (*abort_flag) return false;
        const uint64_t now = globaltimer_ns();
        if (!t0) t0 = now;
        if (now - t0 > kTimeoutNs) {
            *abort_flag = 1;
            report(status, H3B_STATUS_MBAR_TIMEOUT);
            return false;
        }
    }
}

// The exponentials of the two tiles take turns: a warp of tile 0 and the one of
// tile 1 that shares its scheduler, and so its special-function unit.  Left to
// themselves the tiles fall into step, whatever distance they start with: both
// compute exponentials at half the rate, and meanwhile nothing else (64 steps:
// 987 TFLOP/s, with turns 1078).
struct Turn {
    uint64_t *mine, *other;  // null: the other tile is not there
    uint32_t phase;
    volatile int* abort_flag;
    int* status;
    __device__ __forceinline__ bool look() const { return !mine || mbar_try_wait(mine, phase & 1u); }
    __device__ __forceinline__ void take(bool seen) const {
        if (!__all_sync(0xFFFFFFFFu, seen)) await(mine, phase, abort_flag, status);  // (if it gives up, so will the next wait)
        __syncwarp();
    }
    __device__ __forceinline__ void pass() const {
        if (mine && (threadIdx.x & 31) == 0) mbar_arrive(other);
    }
};

// One step of a row: S (64 columns at tS) -> P (bf16, 32 columns at tS), with the
// running maximum and sum.  n: valid keys; sk, sv: factors of the scores (softmax
// scale, log2 e and, for codes, the block's scale) and of the values.  TAIL: not
// all keys are valid.  product_done() waits for the product before, after which O
// may be rescaled; first: there is none.
template <int D, Source SRC, bool TAIL, typename Wait>
__device__ __forceinline__ void softmax_step(Row& st, uint32_t tS, uint32_t tO, bool first, int n, float sk, float sv,
                                             const Wait& product_done, const Turn& turn) {
    uint32_t r[2][32];
    tmem_ld32_async(tS, r[0]);
    tmem_ld32_async(tS + 32, r[1]);
    tmem_ready(r[0]);
    tmem_ready(r[1]);
    const bool seen = turn.look();  // (asked here, answered below)
    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int e = 0; e < 64; e += 2) {
        float y[2] = {__uint_as_float(r[e / 32][e % 32]), __uint_as_float(r[e / 32][e % 32 + 1])};
        if constexpr (TAIL) {
            if (e >= n) y[0] = -INFINITY;
            if (e + 1 >= n) y[1] = -INFINITY;
        }
        mx[(e >> 1) & 3] = max3_nan(mx[(e >> 1) & 3], y[0], y[1]);
    }
    // the step's largest score, NaN if one is
    float top = max3_nan(max3_nan(mx[0], mx[1], mx[2]), mx[3], mx[3]) * sk;
    if (TAIL && n == 0) top = -INFINITY;
    const bool moves = top > st.m + kSlack || (st.m == -INFINITY && top > st.m);
    if (__any_sync(0xFFFFFFFFu, moves)) {
        const float keep = moves ? ex2(st.m - top) : 1.0f;
        if (moves) st.m = top;
        st.l *= keep;
        if (!first) {
            product_done();
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
                uint32_t o[16];
                tmem_ld16(tO + c * 16, o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                tmem_st16(tO + c * 16, o);
            }
        }
    }
    // a NaN or +infinity among the scores makes the row NaN, through its sum
    if (!(top < INFINITY)) st.l = __int_as_float(0x7FC00000);
    const float ref = st.m == -INFINITY ? 0.0f : st.m;
    float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
    turn.take(seen);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        if (c == 1) turn.pass();  // (before the second half of the exponentials)
        uint32_t p[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            float2 x = fma2(make_float2(__uint_as_float(r[c][2 * e]), __uint_as_float(r[c][2 * e + 1])),
                            make_float2(sk, sk), make_float2(-ref, -ref));
            if constexpr (TAIL) {  // behind the product: a scale of zero must not bring a masked key back as NaN
                if (c * 32 + 2 * e >= n) x.x = -INFINITY;
                if (c * 32 + 2 * e + 1 >= n) x.y = -INFINITY;
            }
            x.x = ex2(x.x);
            x.y = ex2(x.y);
            sum[e & 1] = add2(sum[e & 1], x);
            // p is rounded to bf16 for the second product (its sum is not): a relative 2^-8 at most a key
            if constexpr (SRC == kWide) x = mul2(x, make_float2(sv, sv));
            p[e] = pack_bf16x2(x.x, x.y);
        }
        tmem_st16(tS + c * 16, p);
    }
    sum[0] = add2(sum[0], sum[1]);
    st.l += sum[0].x + sum[0].y;
}

// An item is a pair of tiles and a part of the keys; its tiles have the same steps.
struct Item {
    int part, step0, steps;
    bool both;        // tile 1 is there
    uint32_t pair;
};

template <Source SRC>
__device__ __forceinline__ uint32_t pairs_of(const Args& a) {
    return SRC == kWide ? ((uint32_t)a.nq + 1) / 2 * (uint32_t)a.heads : ((uint32_t)a.nq * (uint32_t)a.heads + 1) / 2;
}

template <Source SRC>
__device__ __forceinline__ Item item_of(const Args& a, uint32_t item) {
    Item it;
    const uint32_t pairs = pairs_of<SRC>(a), all = (uint32_t)a.segs;
    it.part = (int)(item / pairs);
    it.pair = item - it.part * pairs;
    it.step0 = (int)(all * it.part / (uint32_t)a.parts);
    it.steps = (int)(all * (it.part + 1) / (uint32_t)a.parts) - it.step0;  // one at least: there are no more parts than steps
    if constexpr (SRC == kWide) {
        const uint32_t row = ((uint32_t)a.nq + 1) / 2;
        it.both = 2 * (it.pair % row) + 1 < (uint32_t)a.nq;
    } else {
        it.both = 2 * it.pair + 1 < (uint32_t)a.nq * (uint32_t)a.heads;
    }
    return it;
}

// Head (within the launch) and query tile of tile t of a pair: query tiles first,
// so that CTAs that run together share a head's keys in L2.
struct Where {
    int h, qt;
};
template <Source SRC>
__device__ __forceinline__ Where where(const Args& a, uint32_t pair, int t) {
    if constexpr (SRC == kWide) {
        const uint32_t row = ((uint32_t)a.nq + 1) / 2, h = pair / row;
        return Where{(int)h, (int)(2 * (pair - h * row)) + t};
    } else {
        const uint32_t id = 2 * pair + t, h = id / (uint32_t)a.nq;
        return Where{(int)h, (int)(id - h * (uint32_t)a.nq)};
    }
}

// Segment `index` of a tile's keys; list: the tile's blocks (kBlocks).  n < 0: an index out of range.
template <Source SRC>
__device__ __forceinline__ Seg segment(const Args& a, const int32_t* list, int index) {
    if (index >= a.segs) return Seg{(int)a.keys, 0};
    int64_t b = index;
    if constexpr (SRC == kBlocks) {
        b = __ldg(list + index);
        if (b < 0 || b * kSeg >= a.keys) return Seg{(int)a.keys, b == -1 ? 0 : -1};
    }
    return Seg{(int)(b * kSeg), (int)min((int64_t)kSeg, a.keys - b * kSeg)};
}
template <Source SRC>
__device__ __forceinline__ const int32_t* list_of(const Args& a, const Where& w) {
    return SRC == kBlocks ? a.blocks + ((int64_t)(a.h0 + w.h) * a.nq + w.qt) * a.topk : nullptr;
}

template <int D, Source SRC>
__global__ void __launch_bounds__(kPairThreads, 1)
    pair_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmO,
                const __grid_constant__ Args a) {
    using L = Smem<D>;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBars);
    uint64_t *kv_full = bars, *kv_empty = bars + 4,  // of the groups
        *s_full = bars + 8, *p_full = bars + 12,     // [tile][buffer]
        *q_full = bars + 16, *q_empty = bars + 18, *pv_done = bars + 20, *o_full = bars + 22, *out_full = bars + 24,  // [tile]
        *drain = bars + 26,
        *out_free = bars + 28,  // the output's place: tile 0 to tile 1, tile 1 to tile 0, tile 0 to itself
        *take = bars + 31;      // [tile][scheduler]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 39);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // the swizzled tiles need the 1024-byte alignment that this declaration asks for
    if (smem_u32(smem) & 1023u) {
        if (threadIdx.x == 0) report(a.status, H3B_STATUS_MBAR_TIMEOUT);
        return;
    }
    if (threadIdx.x == 0) {
        for (int j = 0; j < 4; ++j) {
            mbar_init(kv_full + j, 1);
            mbar_init(kv_empty + j, SRC == kWide ? 2 : 1);  // (kWide: both tiles read a group)
            mbar_init(s_full + j, 1);
            mbar_init(p_full + j, 4);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(q_full + t, 1);
            mbar_init(q_empty + t, 1);
            mbar_init(pv_done + t, 1);
            mbar_init(o_full + t, 1);
            mbar_init(out_full + t, 4);
            mbar_init(drain + t, 1);
        }
        for (int j = 0; j < 3; ++j) mbar_init(out_free + j, 1);
        for (int j = 0; j < 8; ++j) mbar_init(take + j, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    // Groups of loads are numbered through the CTA's steps: group g brings the keys of step g and the values of step
    // g - 2, for one tile (kBlocks, two places each) or for both (kWide, four places).
    if (warp == 8 || warp == 9) {
        // ---------------- MMA issuer of tile t
        if (lane == 0) {
            const int t = warp - 8;
            const uint32_t id_s = idesc(kSeg, false) | (a.scale < 0.0f ? 1u << 13 : 0u);
            const uint32_t id_o = idesc(D, true);
            const uint32_t q0 = desc_k(smem + L::kQ + t * L::kTile), k0 = desc_k(smem + L::kKV),
                           v0 = desc_mn(smem + L::kKV + L::kSegTile);
            const uint32_t tS = tmem + 128 * t, tO = tmem + 256 + 128 * t;
            bool ok = true;
            uint32_t g = 0;                    // groups so far
            uint32_t nq = 0, ns = 0, np = 0;   // this tile's items, scores and products so far
            auto wait = [&](uint64_t* bar, uint32_t phase) { ok = ok && await(bar, phase, abort_flag, a.status); };
            // The products that group g is for: O += P V of step g - 2 (if the tile has that step; fresh, final: its
            // item's first and last) and S = Q K^T of step g (the same; begin, end).  S goes where P of
            // two steps before was, which the product before has read (MMAs run in order)
            auto group = [&](bool output, bool fresh, bool final, bool scores, bool begin, bool end) {
                const uint32_t place = SRC == kWide ? g & 3u : 2 * t + (g & 1u);
                const uint32_t off = place * (L::kGroup >> 4);
                const uint32_t kv_phase = (SRC == kWide ? g >> 2 : g >> 1) & 1u, p_phase = (np >> 1) & 1u;
                uint64_t* const p_bar = p_full + 2 * t + (np & 1u);
                const bool kv_there = mbar_try_wait(kv_full + place, kv_phase);
                const bool p_there = !output || mbar_try_wait(p_bar, p_phase);
                if (!kv_there) wait(kv_full + place, kv_phase);
                if (scores && begin) wait(q_full + t, nq);
                if (output) {
                    const uint32_t buf = np & 1u;
                    if (!p_there) wait(p_bar, p_phase);
                    if (!ok) return;
                    tc_fence_after();
#pragma unroll
                    for (int j = 0; j < kSeg / 16; ++j)
                        mma_ts(tO, tS + 64 * buf + 8 * j, v0 + off + j * (2048 >> 4), id_o, j > 0 || !fresh);
                    umma_commit(pv_done + t);
                    if (final) umma_commit(o_full + t);
                    ++np;
                }
                if (scores) {
                    if (!ok) return;
                    const uint32_t buf = ns & 1u;
                    tc_fence_after();
#pragma unroll
                    for (int j = 0; j < D / 16; ++j)
                        mma_ss(tS + 64 * buf, q0 + (((j / 4) * 16384 + (j % 4) * 32) >> 4),
                               k0 + off + (((j / 4) * L::kSegHalf + (j % 4) * 32) >> 4), id_s, j);
                    umma_commit(s_full + 2 * t + buf);
                    ++ns;
                    if (end) {
                        umma_commit(q_empty + t);
                        ++nq;
                    }
                }
                if (ok) umma_commit(kv_empty + place);
                ++g;
            };
            // steps two and one before: does the tile have them, are they their items' first or last?
            bool has2 = false, has1 = false, first2 = false, first1 = false, last2 = false, last1 = false;
            for (uint32_t item = blockIdx.x; ok && item < a.items; item += gridDim.x) {
                const Item it = item_of<SRC>(a, item);
                const bool has = t == 0 || it.both;
                if (SRC == kBlocks && !has) continue;  // (there are no loads for it)
                for (int i = 0; ok && i < it.steps; ++i) {
                    group(has2, first2, last2, has, i == 0, i + 1 == it.steps);
                    has2 = has1;
                    first2 = first1;
                    last2 = last1;
                    has1 = has;
                    first1 = i == 0;
                    last1 = i + 1 == it.steps;
                }
            }
            if (ok && g > 0) {
                group(has2, first2, last2, false, false, false);
                if (ok) group(has1, first1, last1, false, false, false);
            }
            if (!ok) {
                // no MMA of this thread stays in flight
                umma_commit(drain + t);
                volatile int no_abort = 0;
                mbar_wait(drain + t, 0, &no_abort, nullptr, 100ull * 1000 * 1000);
            }
        }
        __syncwarp();
    } else if (warp == 10 || warp == 11) {
        // ---------------- TMA loads of tile t (keys and values of kWide by the first warp alone), in the order in
        // which the MMAs free their places.  What is not there (a gap in the list, keys behind the last) lies outside
        // the tensor and arrives as zeros
        if (lane == 0) {
            const int t = warp - 10;
            const bool loads = SRC == kBlocks || t == 0;
            bool ok = true;
            uint32_t armed[4] = {0, 0, 0, 0}, nq = 0, g = 0;  // loads so far into each place, items, groups
            // a step's keys are loaded with the values of the step two before it; at < 0: none
            struct Keys {
                int h, at;
            };
            auto load = [&](const Keys& k, const Keys& v) {
                const int place = (int)(SRC == kWide ? g & 3u : 2 * t + (g & 1u));
                uint32_t& n = armed[SRC == kWide ? g & 3u : g & 1u];
                ok = ok && await(kv_empty + place, n + 1, abort_flag, a.status);  // (the first passes at once)
                if (!ok) return;
                uint8_t* dst = smem + L::kKV + place * L::kGroup;
                mbar_expect_tx(kv_full + place, (k.at >= 0 ? L::kSegTile : 0) + (v.at >= 0 ? L::kSegTile : 0));
                ++n;
                ++g;
                if (k.at >= 0) tma_load(dst, &tmK, kv_full + place, k.at, k.h);
                if (v.at >= 0) tma_load(dst + L::kSegTile, &tmV, kv_full + place, v.at, v.h);
            };
            Keys k1{0, -1}, k2{0, -1};  // of the steps one and two before
            for (uint32_t item = blockIdx.x; ok && item < a.items; item += gridDim.x) {
                const Item it = item_of<SRC>(a, item);
                if (t == 1 && !it.both) continue;
                const Where w = where<SRC>(a, it.pair, t);
                const int32_t* list = list_of<SRC>(a, w);
                // (blocks are looked up a step ahead of their load)
                Seg seg = loads ? segment<SRC>(a, list, it.step0) : Seg{0, 0};
                ok = ok && await(q_empty + t, nq + 1, abort_flag, a.status);
                if (!ok) break;
                mbar_expect_tx(q_full + t, L::kTile);
                ++nq;
                tma_load(smem + L::kQ + t * L::kTile, &tmQ, q_full + t, w.qt * kQRows, a.h0 + w.h);
                for (int i = 0; ok && loads && i < it.steps; ++i) {
                    const Seg next = i + 1 < it.steps ? segment<SRC>(a, list, it.step0 + i + 1) : seg;
                    if (seg.n < 0) report(a.status, H3B_STATUS_BAD_INDEX);
                    const Keys k{SRC == kWide ? w.h : a.h0 + w.h, seg.at};
                    load(k, k2);
                    k2 = k1;
                    k1 = k;
                    seg = next;
                }
            }
            // the values of the last two steps
            if (loads && g > 0) {
                load(Keys{0, -1}, k2);
                load(Keys{0, -1}, k1);
            }
            if (!ok) {
                // let the loads in flight land before the CTA exits
                volatile int no_abort = 0;
                for (int j = 0; j < 4; ++j)
                    if (armed[j])
                        mbar_wait(kv_full + (SRC == kWide ? j : 2 * t + j), (armed[j] - 1u) & 1u, &no_abort, nullptr,
                                  100ull * 1000 * 1000);
                if (nq) mbar_wait(q_full + t, (nq - 1u) & 1u, &no_abort, nullptr, 100ull * 1000 * 1000);
            }
        }
        __syncwarp();
    } else {
        // ---------------- softmax and output of tile t, one query row a thread
        const int t = warp >> 2, trow = threadIdx.x & 127;
        const uint32_t at = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tS = tmem + at + 128 * t, tO = tmem + at + 256 + 128 * t;
        const float scale2 = fabsf(a.scale) * kLog2e;
        // this tile's steps and outputs so far, the steps of both
        uint32_t step = 0, outs = 0, shared = 0;
        // items so far with both tiles and with tile 0 alone, which of the two the one before is
        uint32_t pairs = 0, alone = 0;
        bool after_pair = true;
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t phase) {
            return __all_sync(0xFFFFFFFFu, await(bar, phase, abort_flag, a.status)) != 0;
        };
        for (uint32_t item = blockIdx.x; ok && item < a.items; item += gridDim.x) {
            const Item it = item_of<SRC>(a, item);
            const Where u = where<SRC>(a, it.pair, t);
            const int32_t* list = list_of<SRC>(a, u);
            // Each output waits for the one before it on the barrier of that hand-over: an item's second for its first, an
            // item's first for the last of the item before (the CTA's very first passes at once).  One barrier for all of
            // them would not do: a wait sees a phase's parity alone, and tile 1, which skips the items without it, could
            // be two phases off.  A hand-over's next phase needs an output of its waiter in between, so it cannot be here.
            uint64_t* const free_bar = out_free + (t == 1 ? 0 : after_pair ? 1 : 2);
            const uint32_t free_phase = t == 1 ? pairs : (after_pair ? pairs : alone) - 1u;
            if (it.both) ++pairs;
            else ++alone;
            after_pair = it.both;
            if (t == 1 && !it.both) continue;
            Row st{-INFINITY, 0.0f};
            struct Factors {
                int n;
                float sk, sv;
            };
            auto factors = [&](int i) {
                const Seg g = segment<SRC>(a, list, it.step0 + i);
                if (SRC == kBlocks) return Factors{g.n, scale2, 1.0f};
                const int64_t b = (int64_t)(a.h0 + u.h) * (a.cap / kSeg) + it.step0 + i;
                // (the scores' signs: widen_kernel; a cache of one block has its values' scale in the output)
                return Factors{g.n, fabsf(__ldg(a.scales[0] + b)), a.segs == 1 ? 1.0f : __ldg(a.scales[1] + b)};
            };
            Factors ahead = factors(0);
            bool keys = SRC == kWide;  // the part has some
            const bool paired = it.both && a.turns;
            for (int i = 0; ok && i < it.steps; ++i, ++step) {
                const Factors f = ahead;
                if (SRC == kBlocks) keys |= f.n > 0;
                // tile 1 follows tile 0's exponentials of the same step, tile 0 tile 1's of the step before
                const Turn turns{paired ? take + (warp & 3) + 4 * t : nullptr, take + (warp & 3) + 4 * (1 - t),
                                 shared + t - 1u, abort_flag, a.status};
                if (paired) ++shared;
                if (i + 1 < it.steps) ahead = factors(i + 1);
                const int buf = 2 * t + (int)(step & 1u);
                if (!(ok = wait(s_full + buf, step >> 1))) break;
                tc_fence_after();
                const uint32_t tX = tS + 64 * (step & 1u);
                // (a wait cannot tell a phase from the second next: all products but the last are known to be done when
                // S is there, and the next waits for this step's P)
                auto product_done = [&] { ok = wait(pv_done + t, step - 1); };
                const float sk = SRC == kBlocks ? scale2 : scale2 * f.sk;
                if (f.n == kSeg)
                    softmax_step<D, SRC, false>(st, tX, tO, i == 0, f.n, sk, f.sv, product_done, turns);
                else
                    softmax_step<D, SRC, true>(st, tX, tO, i == 0, max(f.n, 0), sk, f.sv, product_done, turns);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + buf);
            }
            if (!ok || !(ok = wait(o_full + t, outs))) break;
            tc_fence_after();
            const int64_t row = (int64_t)u.qt * kQRows + trow;
            const bool split = a.parts > 1;
            float inv = keys ? 1.0f / st.l : 0.0f;
            // (one block: its scale is not rounded with p, whose rounding would be that of every output of a head where
            // there is one token)
            if (SRC == kWide && a.segs == 1) inv *= __ldg(a.scales[1] + (int64_t)(a.h0 + u.h) * (a.cap / kSeg));
            const int64_t slot = ((int64_t)it.part * a.heads + u.h) * a.Sq + row;
            if (split && row < a.Sq)
                *reinterpret_cast<float2*>(a.part_ml + 2 * slot) = make_float2(keys ? fmaxf(st.m, kLowest) : st.m, st.l);
            // the output's place is free when the store before has read it
            if (!split && !(ok = wait(free_bar, free_phase))) break;
            // O: as it is to the join if this is a part of the keys, else through shared memory into whole rows of o
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
                uint32_t r[32];
                tmem_ld32_async(tO + c * 32, r);
                tmem_ready(r);
                if (split) {
                    if (row < a.Sq) {
                        uint4* dst = reinterpret_cast<uint4*>(a.part_o + slot * D + c * 32);
#pragma unroll
                        for (int e = 0; e < 8; ++e) dst[e] = make_uint4(r[4 * e], r[4 * e + 1], r[4 * e + 2], r[4 * e + 3]);
                    }
                } else {
                    uint8_t* half = smem + L::kO + (c / 2) * 16384 + trow * 128;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint32_t o[4];
#pragma unroll
                        for (int f = 0; f < 4; ++f)
                            o[f] = pack_bf16x2(__uint_as_float(r[8 * e + 2 * f]) * inv,
                                               __uint_as_float(r[8 * e + 2 * f + 1]) * inv);
                        *reinterpret_cast<uint4*>(half + ((((c & 1) * 4 + e) ^ (trow & 7)) << 4)) =
                            make_uint4(o[0], o[1], o[2], o[3]);
                    }
                }
            }
            tc_fence_before();
            if (!split) {
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(out_full + t);
                if ((warp & 3) == 0) {
                    if (!(ok = wait(out_full + t, outs))) break;
                    if (lane == 0) {
                        tma_store(&tmO, smem + L::kO, u.qt * kQRows, a.h0 + u.h);
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                        mbar_arrive(out_free + (t == 1 ? 1 : it.both ? 0 : 2));
                    }
                    __syncwarp();
                }
            }
            ++outs;
        }
        // the stores have to be done before the CTA's memory goes
        if (lane == 0 && (warp & 3) == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        __syncwarp();
    }

    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 8)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

// ---------------------------------------------------------------------------
// Rows kernel: few query rows over the cache.  The codes are read once, straight
// into registers, and widened there as the A operand of mma.sync m16n8k16 with
// the query rows as its 8 columns (GROUPS times 8 rows a warp), 16 keys a turn:
//   S^T = K Q^T   thread (g, c) = (lane / 4, lane % 4) holds D / 4 channels of
//                 keys g and g + 8
//   O^T = V^T P^T it holds D / 8 channels of keys 2 c, 2 c + 1, 2 c + 8, 2 c + 9
// (which channel an operand's register stands for is ours to choose), so a load
// is 16 or 8 consecutive codes, and P^T is S^T's accumulators transposed 8 x 8.
//
// Operands are fp16, to which a code widens in fewer instructions than to bf16
// (0x6400 | code + 128 is 1024 + code + 128): the codes are exact; a query row
// is scaled by a power of two that brings its largest element to 2^14 (elements
// are exact down to 2^-28 of it and off by 2^-39 of it below); p is taken 2^11
// times larger and its reference moves at 2^4, so it stays below 2^15 and what
// rounds to zero is below 2^-35 of the largest.  A block's value scale would
// leave that range: each block's output is accumulated apart and joins O with it.
//
// What bounds it is the cache's bytes.  16 keys of 128 channels take about 270
// instructions for 8 rows, 40% of what an SM can issue in the time that HBM
// takes to deliver them.  One row over 131071 tokens of 40 heads: 0.25 ms, 5.3 TB/s.

// Warps of a CTA, each with its own segments: 4, or 8 where that spares the split
// of a short cache and the join (one row over 512 tokens).
constexpr int kRowWarps = 4, kRowWarpsMost = 8;
constexpr float kRowSlack = 4.0f, kRowBias = 11.0f;
// Up to this many rows the rows kernel reads the codes once per 16 rows (from L2
// after the first); beyond, they are widened once for the pair kernel (64 rows
// over 16384 tokens of 40 heads: 190 us and 180; over 60000 of 10: 160 and 162;
// over 512 of 40: 25 and 35; 48 rows over 16384 of 40: 153 and 180).
constexpr int64_t kRowsMost = 64;

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// Codes with their sign bit flipped, bytes 0 and 1 (or 2 and 3) of x -> fp16x2
template <bool HIGH>
__device__ __forceinline__ uint32_t half_codes(uint32_t x) {
    const uint32_t t = __byte_perm(x, 0x64646464u, HIGH ? 0x4342 : 0x4140), base = 0x64806480u;  // 1024 + 128
    const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&t), *reinterpret_cast<const __half2*>(&base));
    return *reinterpret_cast<const uint32_t*>(&d);
}

// CTAs an SM: as many as the registers allow almost without spilling (three instead of
// two: 0.248 ms instead of 0.302 for a row over 131071 tokens of 40 heads).
constexpr int row_ctas(int64_t D, int groups) { return groups == 2 ? 2 : D == 128 ? 3 : 4; }

template <int D, int GROUPS, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, row_ctas(D, GROUPS) * kRowWarps / WARPS)
    rows_kernel(const __grid_constant__ Args a) {
    constexpr int kRows = 8 * GROUPS;
    constexpr int kC = D / 4;     // channels of a thread's keys (scores)
    constexpr int kN = D / 8;     // channels of a thread's keys (output)
    constexpr int kKW = kC / 16;  // uint4 a key
    constexpr int kNW = kN / 4;   // words a key (output)
    using Piece = typename std::conditional<D == 128, uint4, uint2>::type;  // kN codes
    __shared__ float so[WARPS][kRows][D];
    __shared__ float sm[WARPS][kRows], sl[WARPS][kRows];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
    // row groups first: CTAs that run together share a head's codes in L2
    const uint32_t tiles = (uint32_t)((a.Sq + kRows - 1) / kRows);
    const uint32_t rest = blockIdx.x / tiles;
    const int64_t row0 = (int64_t)(blockIdx.x - rest * tiles) * kRows;
    const int part = (int)(rest / (uint32_t)a.H), h = (int)(rest - part * (uint32_t)a.H);
    const int rows = (int)min((int64_t)kRows, a.Sq - row0);

    // this warp's segments: seg0, seg0 + WARPS, .. below seg1
    const int64_t seg1 = a.segs * (part + 1) / a.parts, seg0 = a.segs * part / a.parts + warp;
    const int8_t* kbase = a.codes[0] + ((int64_t)h * a.cap + g) * D + c * kC;
    const int8_t* vbase = a.codes[1] + ((int64_t)h * a.cap + 2 * c) * D + g * kN;
    const float* ks = a.scales[0] + (int64_t)h * (a.cap / kSeg);
    const float* vs = a.scales[1] + (int64_t)h * (a.cap / kSeg);
    uint4 kx[2][kKW];
    Piece vx[4];
    auto fetch = [&](int64_t seg, int turn) {
        const int64_t at = (seg * kSeg + turn * 16) * D;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int w = 0; w < kKW; ++w) kx[t][w] = __ldcs(reinterpret_cast<const uint4*>(kbase + at + t * 8 * D) + w);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            vx[k] = __ldcs(reinterpret_cast<const Piece*>(vbase + at + ((k & 1) + (k & 2) * 4) * D));
    };
    float sk = 0.0f, sv = 0.0f;
    if (seg0 < seg1) {
        fetch(seg0, 0);
        sk = __ldg(ks + seg0);
        sv = __ldg(vs + seg0);
    }

    // Q^T: row g of each group, channels kC c ..
    uint32_t q[GROUPS][kC / 2];
    float factor[GROUPS][2];  // of the scores of rows 2 c, 2 c + 1
#pragma unroll
    for (int r = 0; r < GROUPS; ++r) {
        const uint16_t* src = a.q + (row0 + 8 * r + g) * a.q_ld + h * a.q_hs + c * kC;
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < kC / 8; ++j) {
            uint4 x = make_uint4(0, 0, 0, 0);
            if (8 * r + g < rows) x = *reinterpret_cast<const uint4*>(src + 8 * j);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                q[r][4 * j + e] = w[e];
                top = max(top, max(w[e] & 0x7FFFu, (w[e] >> 16) & 0x7FFFu));
            }
        }
        top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
        top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
        // exponent field of the largest element; 2^(14 - exponent) as long as that is a number, 1 beside an
        // infinity or NaN
        const int e = max((int)(top >> 7), 40);
        const float up = e == 255 ? 1.0f : __int_as_float((127 + 14 + 127 - e) << 23);
        const float down = e == 255 ? 1.0f : __int_as_float((127 - 14 - 127 + e) > 0 ? (e - 14) << 23 : 0);
#pragma unroll
        for (int j = 0; j < kC / 2; ++j) q[r][j] = pack_half2(bf16_lo(q[r][j]) * up, bf16_hi(q[r][j]) * up);
#pragma unroll
        for (int k = 0; k < 2; ++k)
            factor[r][k] = a.scale * kLog2e * __shfl_sync(0xFFFFFFFFu, down, (2 * c + k) * 4);
    }

    float o[GROUPS][kN / 2][4], m[GROUPS][2], l[GROUPS][2];
#pragma unroll
    for (int r = 0; r < GROUPS; ++r) {
#pragma unroll
        for (int j = 0; j < kN / 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[r][j][e] = 0.0f;
        m[r][0] = m[r][1] = -INFINITY;
        l[r][0] = l[r][1] = 0.0f;
    }

    for (int64_t seg = seg0; seg < seg1; seg += WARPS) {
        const float fk = sk, fv = sv;
        const int valid = (int)min((int64_t)kSeg, a.keys - seg * kSeg);
        const bool more = seg + WARPS < seg1;
        if (more) {
            sk = __ldg(ks + seg + WARPS);
            sv = __ldg(vs + seg + WARPS);
        }
        float os[GROUPS][kN / 2][4];  // this block's output, without its scale
#pragma unroll
        for (int r = 0; r < GROUPS; ++r)
#pragma unroll
            for (int j = 0; j < kN / 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) os[r][j][e] = 0.0f;
#pragma unroll 1
        for (int turn = 0; turn < kSeg / 16; ++turn) {
            uint32_t kc[2][kC / 4], vc[4][kNW];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int w = 0; w < kC / 4; ++w) kc[t][w] = reinterpret_cast<const uint32_t*>(kx[t])[w] ^ 0x80808080u;
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int w = 0; w < kNW; ++w) vc[k][w] = reinterpret_cast<const uint32_t*>(&vx[k])[w] ^ 0x80808080u;
            if (turn + 1 < kSeg / 16) fetch(seg, turn + 1);
            else if (more) fetch(seg + WARPS, 0);
            float s[GROUPS][4];
#pragma unroll
            for (int r = 0; r < GROUPS; ++r) s[r][0] = s[r][1] = s[r][2] = s[r][3] = 0.0f;
#pragma unroll
            for (int j = 0; j < kC / 4; ++j) {
                const uint32_t a0 = half_codes<false>(kc[0][j]), a1 = half_codes<false>(kc[1][j]),
                               a2 = half_codes<true>(kc[0][j]), a3 = half_codes<true>(kc[1][j]);
#pragma unroll
                for (int r = 0; r < GROUPS; ++r) mma_16816(s[r], a0, a1, a2, a3, q[r][2 * j], q[r][2 * j + 1]);
            }
            // s[r][2 t + k]: key g + 8 t, row 2 c + k
            const int left = valid - turn * 16 - g;
            bool moves = false;
#pragma unroll
            for (int r = 0; r < GROUPS; ++r)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[r][e] = (e < 2 ? 0 : 8) < left ? s[r][e] * (fk * factor[r][e & 1]) : -INFINITY;
                    moves |= s[r][e] > m[r][e & 1] + kRowSlack || (m[r][e & 1] == -INFINITY && s[r][e] > -INFINITY);
                }
            if (__any_sync(0xFFFFFFFFu, moves)) {
#pragma unroll
                for (int r = 0; r < GROUPS; ++r) {
                    float keep[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        float top = fmaxf(s[r][k], s[r][2 + k]);
#pragma unroll
                        for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, off));
                        const float to = fmaxf(m[r][k], top);
                        keep[k] = to == m[r][k] ? 1.0f : ex2(m[r][k] - to);
                        m[r][k] = to;
                        l[r][k] *= keep[k];
                    }
#pragma unroll
                    for (int j = 0; j < kN / 2; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            o[r][j][e] *= keep[e & 1];
                            os[r][j][e] *= keep[e & 1];
                        }
                }
            }
            uint32_t p[GROUPS][2];
#pragma unroll
            for (int r = 0; r < GROUPS; ++r) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float ref = m[r][e & 1] == -INFINITY ? 0.0f : m[r][e & 1] - kRowBias;
                    s[r][e] = ex2(s[r][e] - ref);
                    l[r][e & 1] += s[r][e];
                }
                // p is rounded to fp16 for the second product (its sum is not): a relative 2^-11 at most a key
                p[r][0] = transpose_8x8(pack_half2(s[r][0], s[r][1]));
                p[r][1] = transpose_8x8(pack_half2(s[r][2], s[r][3]));
            }
            // tile j has channels kN g + 2 j and 2 j + 1 of this thread, whose keys are bytes of four words
#pragma unroll
            for (int w = 0; w < kNW; ++w)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int sel = half ? 0x7362 : 0x5140;
                    const uint32_t x = __byte_perm(vc[0][w], vc[1][w], sel), y = __byte_perm(vc[2][w], vc[3][w], sel);
                    const uint32_t a0 = half_codes<false>(x), a1 = half_codes<true>(x), a2 = half_codes<false>(y),
                                   a3 = half_codes<true>(y);
#pragma unroll
                    for (int r = 0; r < GROUPS; ++r) mma_16816(os[r][2 * w + half], a0, a1, a2, a3, p[r][0], p[r][1]);
                }
        }
#pragma unroll
        for (int r = 0; r < GROUPS; ++r)
#pragma unroll
            for (int j = 0; j < kN / 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[r][j][e] = fmaf(os[r][j][e], fv, o[r][j][e]);
    }
    // the warps' parts meet in shared memory
#pragma unroll
    for (int r = 0; r < GROUPS; ++r)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int row = 8 * r + 2 * c + k;
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) l[r][k] += __shfl_xor_sync(0xFFFFFFFFu, l[r][k], off);
            if (g == 0) {
                sm[warp][row] = m[r][k];
                sl[warp][row] = l[r][k];
            }
            if (row < rows) {
#pragma unroll
                for (int j = 0; j < kN / 2; ++j)
                    *reinterpret_cast<float2*>(&so[warp][row][kN * g + 2 * j]) = make_float2(o[r][j][k], o[r][j][2 + k]);
            }
        }
    __syncthreads();
    for (int e = threadIdx.x; e < rows * (D / 2); e += 32 * WARPS) {
        const int r = e / (D / 2), ch = 2 * (e % (D / 2));
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top = fmaxf(top, sm[w][r]);
        const float ref = top == -INFINITY ? 0.0f : top;
        float total = 0.0f, x = 0.0f, y = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float f = ex2(sm[w][r] - ref);
            total += f * sl[w][r];
            x += f * so[w][r][ch];
            y += f * so[w][r][ch + 1];
        }
        if (a.parts > 1) {
            const int64_t slot = ((int64_t)part * a.H + h) * a.Sq + row0 + r;
            *reinterpret_cast<float2*>(a.part_o + slot * D + ch) = make_float2(x, y);
            if (ch == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * slot) = make_float2(fmaxf(top, kLowest), total);
        } else {
            const float inv = 1.0f / total;
            *reinterpret_cast<uint32_t*>(a.o + (row0 + r) * a.o_ld + h * a.o_hs + ch) = pack_bf16x2(x * inv, y * inv);
        }
    }
}

// Join of the parts of a split: o = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s.
// One CTA a row and head; its warps take the parts in turn.
template <int D>
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ Args a) {
    constexpr int E = D / 32;
    __shared__ float so[4][D], sl[4];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t id = blockIdx.x, step = a.Sq * a.heads;
    const int h = a.h0 + (int)(id / a.Sq);
    const int64_t row = id % a.Sq;
    float m = -INFINITY;
    for (int s = lane; s < a.parts; s += 32) m = fmaxf(m, a.part_ml[2 * (s * step + id)]);
#pragma unroll
    for (int off = 16; off; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, off));
    const float ref = m == -INFINITY ? 0.0f : m;
    float l = 0.0f, o[E] = {};
#pragma unroll 4
    for (int s = warp; s < a.parts; s += 4) {
        const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * (s * step + id));
        const float w = ex2(ml.x - ref);
        l += w * ml.y;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] += w * a.part_o[(s * step + id) * D + lane * E + e];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) so[warp][lane * E + e] = o[e];
    if (lane == 0) sl[warp] = l;
    __syncthreads();
    if (threadIdx.x < D / 2) {
        const int ch = 2 * threadIdx.x;
        const float total = (sl[0] + sl[1]) + (sl[2] + sl[3]);
        const float inv = m == -INFINITY ? 0.0f : 1.0f / total;
        float x[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) x[e] = ((so[0][ch + e] + so[1][ch + e]) + (so[2][ch + e] + so[3][ch + e])) * inv;
        *reinterpret_cast<uint32_t*>(a.o + row * a.o_ld + h * a.o_hs + ch) = pack_bf16x2(x[0], x[1]);
    }
}

// o = 0 where there is no key at all, 8 channels a thread.
__global__ void __launch_bounds__(256) zero_kernel(Args a, int per_head, int64_t pieces) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= pieces) return;
    const int64_t row = i / per_head;
    *reinterpret_cast<uint4*>(a.o + row / a.H * a.o_ld + row % a.H * a.o_hs + i % per_head * 8) = make_uint4(0, 0, 0, 0);
}

// Codes of some heads (each `per` pieces of 16 from `stride` pieces apart) -> bf16, K or V by blockIdx.y.  A key
// scale's sign goes into the codes (2^block_log2 pieces share a scale): the maximum of a block's scores is taken
// before its scale, which must not turn their order.  (Turning the scores there costs the long kernel 2%.)
__global__ void __launch_bounds__(256) widen_kernel(const int8_t* __restrict__ kq, const int8_t* __restrict__ vq,
                                                    const float* __restrict__ ks, int64_t stride, int64_t per,
                                                    int64_t pieces, int block_log2,
                                                    uint16_t* __restrict__ k, uint16_t* __restrict__ v) {
    const uint4* src = reinterpret_cast<const uint4*>(blockIdx.y ? vq : kq);
    uint4* dst = reinterpret_cast<uint4*>(blockIdx.y ? v : k);
    uint4 x[4];
    uint32_t sign[4];
    const int64_t first = (int64_t)blockIdx.x * 1024 + threadIdx.x;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const int64_t i = first + p * 256;
        if (i >= pieces) break;
        const int64_t at = i / per * stride + i % per;
        x[p] = __ldg(src + at);
        sign[p] = blockIdx.y == 0 && __ldg(ks + (at >> block_log2)) < 0.0f ? 0x80008000u : 0u;
    }
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const int64_t i = first + p * 256;
        if (i >= pieces) break;
        const uint32_t w[4] = {x[p].x, x[p].y, x[p].z, x[p].w};
#pragma unroll
        for (int e = 0; e < 2; ++e)
            dst[2 * i + e] = make_uint4(
                codes_to_bf16x2(w[2 * e], 0x4140) ^ sign[p], codes_to_bf16x2(w[2 * e], 0x4342) ^ sign[p],
                codes_to_bf16x2(w[2 * e + 1], 0x4140) ^ sign[p], codes_to_bf16x2(w[2 * e + 1], 0x4342) ^ sign[p]);
    }
}

// [tokens, heads, D] bf16 as boxes of `rows` tokens of a head (see tma_load).
static int make_map(CUtensorMap* map, const void* p, int64_t n, int H, int64_t D, int64_t ld, int64_t hs, int rows) {
    PFN_encodeTiled enc = encode_fn();
    if (!enc) return set_error(H3B_ERR_CUDA, "cuTensorMapEncodeTiled unavailable (driver too old?)");
    cuuint64_t dims[4] = {64, (cuuint64_t)n, (cuuint64_t)(D / 64), (cuuint64_t)H};
    cuuint64_t strides[3] = {(cuuint64_t)ld * 2, 128, (cuuint64_t)hs * 2};
    cuuint32_t box[4] = {64, (cuuint32_t)rows, (cuuint32_t)(D / 64), 1};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(p), dims, strides, box, estr,
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

// Parts that the keys of every row tile are split into.  All pairs of tiles take
// about as long, so the time is the number of rounds of a pair an SM times a
// part's steps plus what a pair spends besides (about four steps); a join costs
// about four more.
static int64_t parts_of(bool cache, int64_t nq, int64_t heads, int64_t steps) {
    int64_t best = 1, best_cost = 0;
    for (int64_t n = 1; n <= 64 && (n == 1 || n <= steps); ++n) {
        const int64_t pairs = (cache ? cdiv(nq, 2) * heads : cdiv(nq * heads, 2)) * n;
        const int64_t cost = cdiv(pairs, sm_count()) * (cdiv(steps, n) + 4) + (n > 1 ? 4 : 0);
        if (n == 1 || cost < best_cost) best = n, best_cost = cost;
    }
    return best;
}

// The same for the rows kernel: rounds of the CTAs that fit, whose warps take a
// segment each at a time, plus about one segment's time for the rest of a CTA.
static int64_t row_parts_of(int64_t tiles, int64_t segs, int ctas) {
    int64_t best = 1, best_cost = 0;
    for (int64_t n = 1; n <= 64 && (n == 1 || n <= cdiv(segs, kRowWarps)); ++n) {
        const int64_t cost = cdiv(tiles * n, ctas * sm_count()) * (cdiv(segs, n * kRowWarps) + 1) + (n > 1 ? 2 : 0);
        if (n == 1 || cost < best_cost) best = n, best_cost = cost;
    }
    return best;
}

struct Plan {
    bool rows;               // the rows kernel
    int warps;               // of its CTAs
    int64_t heads;           // heads a launch (and of the widened copy)
    int64_t parts;           // of the keys
    int64_t join_at, bytes;  // in the workspace
};

// of widened heads at a time (one head at least): 256 rows over 16384 tokens of 40 heads 211 us, with 256 MiB 227
constexpr int64_t kWideBytes = 512ll << 20;

static Plan plan(bool cache, int64_t Sq, int64_t H, int64_t D, int64_t segs) {
    Plan p{false, 0, H, 1, 0, 0};
    if (segs == 0) return p;
    if (cache && Sq <= kRowsMost) {
        p.rows = true;
        const int groups = Sq <= 8 ? 1 : 2;
        p.parts = row_parts_of(cdiv(Sq, 8 * groups) * H, segs, row_ctas(D, groups));
        p.warps = groups == 1 && p.parts <= 2 && segs > kRowWarps && H <= sm_count() ? kRowWarpsMost : kRowWarps;
        if (p.warps == kRowWarpsMost) p.parts = 1;
        p.bytes = p.parts > 1 ? p.parts * H * Sq * (D + 2) * 4 : 0;
        return p;
    }
    const int64_t nq = cdiv(Sq, kQRows);
    const int64_t head = cache ? 2 * segs * kSeg * D * 2 : 0;
    if (H * head > kWideBytes) {
        // as few launches as that allows, of about as many heads each (16 and 4 heads: 1.05 ms, 10 and 10: 0.85)
        const int64_t most = kWideBytes / head > 0 ? kWideBytes / head : 1;
        p.heads = cdiv(H, cdiv(H, most));
    }
    p.parts = parts_of(cache, nq, p.heads, segs);
    p.join_at = p.heads * head;
    p.bytes = p.join_at + (p.parts > 1 ? p.parts * p.heads * Sq * (D + 2) * 4 : 0);
    return p;
}

template <int D, Source SRC>
static int launch_pairs(Args a, const uint16_t* const (&kv)[2], const int64_t (&ld)[2], const int64_t (&hs)[2],
                        cudaStream_t s) {
    CUtensorMap q, k, v, o;
    if (int rc = make_map(&q, a.q, a.Sq, a.H, D, a.q_ld, a.q_hs, kQRows)) return rc;
    if (int rc = make_map(&o, a.o, a.Sq, a.H, D, a.o_ld, a.o_hs, kQRows)) return rc;
    const int n = SRC == kBlocks ? a.H : a.heads;
    if (int rc = make_map(&k, kv[0], a.keys, n, D, ld[0], hs[0], kSeg)) return rc;
    if (int rc = make_map(&v, kv[1], a.keys, n, D, ld[1], hs[1], kSeg)) return rc;
    const int64_t items = (SRC == kWide ? cdiv(a.nq, 2) * a.heads : cdiv(a.nq * a.heads, 2)) * a.parts;
    a.items = (uint32_t)items;
    // Turns pay where items are long (64 steps: 1.02 ms instead of 1.11) and cost where a tile's output keeps the
    // other waiting every few steps (8 steps: 1.68 ms instead of 1.59).
    a.turns = a.segs / a.parts >= 24;
    H3B_CUDA_TRY(cudaFuncSetAttribute(pair_kernel<D, SRC>, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<D>::kBytes));
    const int64_t grid = items < sm_count() ? items : sm_count();
    pair_kernel<D, SRC><<<(unsigned)grid, kPairThreads, Smem<D>::kBytes, s>>>(q, k, v, o, a);
    if (a.parts > 1) join_kernel<D><<<(unsigned)(a.Sq * a.heads), 128, 0, s>>>(a);
    H3B_CUDA_TRY(cudaGetLastError());
    return H3B_OK;
}

template <int D>
static int launch_all(Args& a, bool cache, const Plan& p, char* ws, cudaStream_t s) {
    a.part_o = reinterpret_cast<float*>(ws + p.join_at);
    a.part_ml = a.part_o + (p.parts > 1 ? p.parts * p.heads * a.Sq * D : 0);
    a.parts = (int)p.parts;
    a.heads = a.H;
    if (p.rows) {
        if (p.warps == kRowWarpsMost) rows_kernel<D, 1, kRowWarpsMost><<<(unsigned)a.H, 32 * kRowWarpsMost, 0, s>>>(a);
        else if (a.Sq <= 8) rows_kernel<D, 1, kRowWarps><<<(unsigned)(a.H * p.parts), 32 * kRowWarps, 0, s>>>(a);
        else rows_kernel<D, 2, kRowWarps><<<(unsigned)(cdiv(a.Sq, 16) * a.H * p.parts), 32 * kRowWarps, 0, s>>>(a);
        if (p.parts > 1) join_kernel<D><<<(unsigned)(a.Sq * a.H), 128, 0, s>>>(a);
        H3B_CUDA_TRY(cudaGetLastError());
        return H3B_OK;
    }
    if (!cache) return launch_pairs<D, kBlocks>(a, a.kv, a.kv_ld, a.kv_hs, s);
    const int64_t rows = a.segs * kSeg;
    uint16_t* const k = reinterpret_cast<uint16_t*>(ws);
    for (int64_t h = 0; h < a.H; h += p.heads) {
        const int64_t n = a.H - h < p.heads ? a.H - h : p.heads;
        uint16_t* const v = k + n * rows * D;
        const int64_t pieces = n * rows * D / 16;
        widen_kernel<<<dim3((unsigned)cdiv(pieces, 4 * 256), 2), 256, 0, s>>>(
            a.codes[0] + h * a.cap * D, a.codes[1] + h * a.cap * D, a.scales[0] + h * (a.cap / kSeg), a.cap * D / 16,
            rows * D / 16, pieces, D == 128 ? 9 : 8, k, v);
        a.h0 = (int)h;
        a.heads = (int)n;
        const int64_t ld[2] = {D, D}, hs[2] = {rows * D, rows * D};
        const uint16_t* const kv[2] = {k, v};
        if (int rc = launch_pairs<D, kWide>(a, kv, ld, hs, s)) return rc;
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
    if (a.keys == 0) segs = 0;
    a.segs = segs;
    a.nq = cdiv(a.Sq, kQRows);
    const Plan p = plan(cache, a.Sq, a.H, D, segs);
    H3B_REQUIRE(a.nq * a.H * p.parts < (1ll << 28) && a.Sq * a.H < (1ll << 31), "%s: too many row tiles", who);
    H3B_REQUIRE(p.bytes == 0 || (ws && aligned(ws, 256) && ws_bytes >= p.bytes),
                "%s: workspace of %lld bytes (256-byte aligned), %lld needed", who, (long long)ws_bytes, (long long)p.bytes);
    DeviceStatus ds;
    if (int rc = device_status(&ds)) return rc;
    a.status = ds.word;
    if (segs == 0) {
        const int64_t pieces = a.Sq * a.H * D / 8;
        zero_kernel<<<(unsigned)cdiv(pieces, 256), 256, 0, s>>>(a, (int)(D / 8), pieces);
        H3B_CUDA_TRY(cudaGetLastError());
        return H3B_OK;
    }
    return D == 128 ? launch_all<128>(a, cache, p, static_cast<char*>(ws), s)
                    : launch_all<64>(a, cache, p, static_cast<char*>(ws), s);
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
    H3B_REQUIRE(topk >= 0 && topk <= (1ll << 25) && H > 0 && H <= 65535, "h3b_block_sparse_attn: topk=%lld heads=%lld out of range",
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
