// hkv_window.cu -- attention of several new tokens per slot over the paged cache
// (prompts, refreshed windows): row i of a slot sees rows [0, used + i].
//
//   s_t = (q . c_t) 2^eK scale log2(e),  w_t = 2^(s_t + eV - m),
//   o   = sum_t w_t c_t,                 out = o / sum_t w_t 2^-eV
//
// with codes c (F16 values in an F16 cache: eK = eV = 0) and m the row's running bound
// of s_t + eV over the keys that it sees; one pass over them.  V's exponent belongs to
// the weight: a row's weights are then at most 1 whatever the exponents are, and keep
// their bits by what a key adds to the row's output, its V as well as its logit.
//
// One CTA takes up to 64 tokens x the 4 query heads of a KV head, as two M = 128
// tiles (row = 4 token + head), so that a key is read and converted once for 256
// rows, and a run of 128-key blocks.  Both products run on the tensor cores
// (tcgen05, F32 accumulators in TMEM); codes are exact in F16, so K and V enter
// without error.
//   warps 0-7, 8-15 softmax of M tile 0 / 1, two threads a row (64 of a block's keys
//                   each): S from TMEM, the weights back into S's columns as the next
//                   product's A operand
//   warps 16-20     converters: 16-byte pieces of the pages to F16 operand tiles
//   warp 21         exponents of each block, and K as it is where q is in E4M3 parts
//   warps 22, 23    one thread each issues the products of an M tile; while one tile's
//                   softmax runs, the other tile's products do
//
// BF16 tensors on an 8-bit cache: q has 8 significant bits, two E4M3 numbers of 4
// (with a power of two per row), so q K^T is two E4M3 products at twice the F16 rate
// and K goes from its pages to shared memory by bulk copies, unconverted: a page's
// code block is the 128-byte-swizzled operand tile already.
// F32 tensors: q and the weights in two F16 parts each, hi + lo, which keeps 22
// bits and doubles the products.  F16 and BF16 tensors: one part.
//
// What bounds it: the chain S, softmax, P, O of a block, which the two tiles of a CTA
// take in turns; tensor pipe, exponentials and issue slots are each under half.  8 KV
// heads, 8-bit cache: a BF16 prompt of 8100 605-645 us by its data (0.55-0.51 of the
// measured bf16 rate), of F16 695, of F32 1033; 8 F32 windows of 4-1024 behind 584-4000 466 us
// (0.51 of the rate for the doubled products; the softmax's longer chain and the moves of
// o weigh most); 37 behind 770 16.7 us (launch, one block's chain, the join).  On an F16
// cache, whose K and V the converters bring through registers at twice the bytes: the
// prompt 1028 us in BF16 or F16, 1268 in F32.
//
// The rescaling of o when the bound m moves is put off until a row passes it by
// 2^kSlack (weights up to 2^kSlack then enter the product); o is rescaled in TMEM
// by the softmax warps, rarely after the first blocks.
//
// Non-finite V values are zeroed in the operand tiles, since 0 * inf would reach
// rows that do not see them; a CTA that met one adds them to the rows that do see
// them at its end, from the blocks that it marked (a prompt of 6000 with one such
// value 2.4 ms, of 0.38 without; 34 with all of V read again).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

#include "hkv_device.cuh"
#include "hkv_e4m3.cuh"
#include "hkv_internal.h"
#include "hkv_tcgen05.cuh"

namespace hkv {
namespace {

using namespace dev;

constexpr int kWhereWindow = 8;
constexpr int kDtypeF32 = 0;
constexpr int kDtypeF16 = 1;

constexpr int kKeys = kWindowKeys;      // keys of a block
constexpr int kBlockPages = kKeys / kPageTokens;
constexpr int kTile = 128;              // rows of an M tile: 32 tokens x 4 heads
constexpr int kTileTokens = kTile / kGqa;
constexpr int kTileBytes = 128 * 128 * 2;   // an F16 operand tile (q rows, keys)
constexpr int kCodeTileBytes = 128 * 128;   // an E4M3 one
static_assert(kKeys == 128 && kTile == 128, "operand tiles are 128 x 128");
constexpr int kTileThreads = 256;       // softmax threads of an M tile
constexpr int kSoftmaxThreads = 2 * kTileThreads;
constexpr int kConvertThreads = 160;
constexpr int kScaleWarp = 21;
constexpr int kIssuer = 22;
constexpr int kThreads = 768;
// Registers of a thread: the launch gives 80 to each, the softmax takes what the
// other two of the six warpgroups leave.
constexpr int kSoftmaxRegs = 88;
constexpr int kOtherRegs = 64;
static_assert(4 * kSoftmaxRegs + 2 * kOtherRegs == 6 * 80, "the shares add up to the launch's registers");
constexpr float kSlack = 8.f;
// A bound is the rounded largest logit: beyond this size it may lie so far from the exact
// one that a weight leaves F16.  There the logits are rounded before the bound is
// subtracted, as a plain F32 softmax rounds them.
constexpr float kHuge = 1 << 23;
constexpr int kShift = 7;               // weights enter 2^7 larger: at most 2^15 in F16
// F32 tensors: blocks after which o moves from TMEM to the row's place in `out` (or in
// the part) and is added there in F32.  The tensor cores cut their sums instead of
// rounding them: each of a block's 16 products takes about 2^-24 of o away, always
// towards zero, 1e-5 of it over 4000 keys.  Eight ragged windows (1024 keys on average
// behind 2034): error 5.7e-6 and 391 us without, 2.5e-6 and 432 us every 8 blocks,
// 1.5e-6 and 461 us every 4.
constexpr int kDrainBlocks = 4;
// V exponents this far below the largest so far: a weight of such a page may underflow in
// F32 though its key weighs, so the sum of the weights is formed apart.  At less, terms
// down to 2^-50 of a row's largest enter it.
constexpr int kFar = 80;
// The least exponent of a row of q in E4M3 parts: with K's least, -100, the factor of a
// logit stays a normal float, as masked logits (-inf) need it.  Smaller rows round to
// multiples of 2^-30, F16 ones to 2^-25.
constexpr int kQExpMin = -20;

// What the softmax needs of a page.
struct alignas(16) PageScale {
    float k;      // scale * log2(e) * 2^eK
    float v_exp;  // eV
    float shift;  // of the weights' exponent: kShift + eV
    float back;   // 2^-(kShift + eV): from weights to terms of the sum; 0 in a far block
};
struct BlockScale {
    PageScale page[kBlockPages];
    int far;      // some eV is more than kFar below the largest so far
};

struct Control {
    uint64_t q_full, s_full[2], o_full[2];
    uint64_t p_full[2][2];      // of a tile: weights of keys 0-31 and 64-95 of the block, and of the others
    uint64_t k_full[3], k_empty[3], v_full[3], v_empty[3];
    uint64_t turn[2];           // of the issuers: a phase a block
    uint64_t drained[2];        // after a wait that ran out: no product in flight
    uint32_t tmem;
    uint32_t odd_v;             // blocks, modulo 32, in which a V value that is not finite was met
    // One region per M tile: the tiles go through their blocks without a barrier between
    // them, so what a tile writes must not lie over what the other may still read.
    union TileRows {
        int q_exp[kTile];             // of a row of q in E4M3 parts
        float half[2][kTile];         // of a block, the bound of a row by each of its threads; l at the end
    } rows[2];
};
static_assert(sizeof(Control) % 16 == 0, "the scales follow it");
static_assert(sizeof(Control::TileRows) == 2 * kTile * sizeof(float), "a tile's exponents lie over its own halves");

template <typename T, bool kE4m3>
struct Shape {
    static constexpr bool kSplit = sizeof(T) == 4;
    static constexpr bool kCodeK = kE4m3 && std::is_same<T, __nv_bfloat16>::value;
    static constexpr int kParts = kSplit || kCodeK ? 2 : 1;  // of q
    // F32: the products of half a block's weights start while the other half's are
    // formed (8100 tokens: 1033 us, 1086 without; on an F16 cache, which waits for its
    // converters, 1265 and 1245); a 16-bit block's softmax is too short for that to pay for
    // its second store and barrier (8 ragged windows: BF16 279 us, 283 with; 8100 tokens of
    // F16 694 and 716).
    static constexpr bool kEarly = kSplit;
    static constexpr int kQPart = kCodeK ? kCodeTileBytes : kTileBytes;
    static constexpr int kKTile = kCodeK ? kCodeTileBytes : kTileBytes;
    static constexpr int kKSlots = kSplit ? 1 : kCodeK ? 3 : 2;
    static constexpr int kVSlots = kSplit ? 2 : 3;
    // Blocks whose scales are kept.  Those of block j are written once the products of
    // q and K of block j - kKSlots are done, when a softmax may still be at that block.
    static constexpr int kScaleSlots = 2 * kKSlots;
    static constexpr int kQBytes = 2 * kParts * kQPart;
    static constexpr int kControl = kQBytes + kKSlots * kKTile + kVSlots * kTileBytes;  // its offset
    static constexpr int kSmem = kControl + sizeof(Control) + kScaleSlots * sizeof(BlockScale);
    static_assert(kSmem <= 227 * 1024, "operands exceed shared memory");
};

__device__ __forceinline__ void record(DeviceError *err, int code, int a, int b) {
    if (atomicCAS(&err->code, 0, code) == 0) {
        err->where = kWhereWindow;
        err->a = a;
        err->b = b;
    }
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t half2_sum(uint32_t a, uint32_t b) {
    const __half2 h = __hadd2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 half2_floats(uint32_t u) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&u));
}
__device__ __forceinline__ void st_shared16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void st_shared8(uint32_t addr, uint32_t a, uint32_t b) {
    asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(addr), "r"(a), "r"(b) : "memory");
}
// L2 policy of K, which the CTAs of other query tiles read again.
__device__ __forceinline__ uint64_t keep_policy() {
    uint64_t policy;
    asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(policy));
    return policy;
}
__device__ __forceinline__ void load8(const float *p, float (&x)[8]) {
    const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void load8(const __half *p, float (&x)[8]) {
    const uint4 u = *reinterpret_cast<const uint4 *>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = half2_floats(w[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void load8(const __nv_bfloat16 *p, float (&x)[8]) {
    const uint4 u = *reinterpret_cast<const uint4 *>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void store4(float *p, const float *x) {
    *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void store4(__half *p, const float *x) {
    *reinterpret_cast<uint2 *>(p) = make_uint2(half2_bits(x[0], x[1]), half2_bits(x[2], x[3]));
}
__device__ __forceinline__ void store4(__nv_bfloat16 *p, const float *x) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
    *reinterpret_cast<uint2 *>(p) =
        make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}

// 16 dims of a row, held by each of four neighbouring lanes, to 4 dims of the four rows:
// o[4 r ..] is then row r's dims 4 j .. 4 j + 3 in lane j of the four.  Rows r are the
// four heads of a token, so an access is 64 bytes of each instead of 16 of 32 rows.
__device__ __forceinline__ void four_rows(float (&o)[16], int lane) {
#pragma unroll
    for (int step = 1; step < 4; step *= 2) {
        const bool up = (lane & step) != 0;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if ((r & step) == 0) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float &a = o[4 * r + k], &b = o[4 * (r + step) + k];
                    const float got = __shfl_xor_sync(0xffffffffu, up ? a : b, step);
                    a = up ? got : a;
                    b = up ? b : got;
                }
            }
        }
    }
}
// What the four lanes of a token hold of x, by row.
__device__ __forceinline__ float4 of_rows(float x, int lane) {
    const int from = lane & ~3;
    return make_float4(__shfl_sync(0xffffffffu, x, from), __shfl_sync(0xffffffffu, x, from + 1),
                       __shfl_sync(0xffffffffu, x, from + 2), __shfl_sync(0xffffffffu, x, from + 3));
}
__device__ __forceinline__ float row_of(const float4 &x, int r) {
    return r == 0 ? x.x : r == 1 ? x.y : r == 2 ? x.z : x.w;
}
// o += scale * s, where the scale is not 0.
__device__ __forceinline__ void plus4(float *o, const float4 &s, float scale) {
    o[0] = scale != 0.f ? fmaf(s.x, scale, o[0]) : o[0];
    o[1] = scale != 0.f ? fmaf(s.y, scale, o[1]) : o[1];
    o[2] = scale != 0.f ? fmaf(s.z, scale, o[2]) : o[2];
    o[3] = scale != 0.f ? fmaf(s.w, scale, o[3]) : o[3];
}

// *p += x in L2, and a load from there.
__device__ __forceinline__ void add_at(float *p, const float *x) {
    asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1,%2,%3,%4};" ::"l"(p), "f"(x[0]), "f"(x[1]), "f"(x[2]),
                 "f"(x[3])
                 : "memory");
}
__device__ __forceinline__ float4 load_at(const float *p) {
    return __ldcg(reinterpret_cast<const float4 *>(p));
}

// A wait of one role.  One that runs out is recorded and ends its role (a softmax warp
// still goes to its barriers); the waits that depend on it run out in turn, and the CTA leaves.
// The threads sleep in try_wait (20 us at a time), so that they leave the issue
// slots to the warps that work.
__device__ __forceinline__ bool try_wait_long(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(20000u)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool wait_for(uint64_t *bar, uint32_t parity, DeviceError *err) {
    const uint32_t at = smem_u32(bar);
    if (try_wait_long(at, parity)) {
        return true;
    }
    const long long t0 = clock64();
    while (clock64() - t0 < kWaitBudgetCycles) {
        if (try_wait_long(at, parity)) {
            return true;
        }
    }
    record(err, kErrTimeout, static_cast<int>(blockIdx.x), static_cast<int>(threadIdx.x));
    return false;
}

// Barrier of the two warps that share rows (w and w + 4): ids 1 .. 8.
__device__ __forceinline__ void pair_barrier(int warp) {
    asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp >> 3) * 4 + (warp & 3)) : "memory");
}

// Barrier of an M tile's softmax threads.
__device__ __forceinline__ void tile_barrier(int i) {
    asm volatile("bar.sync %0, 256;" ::"r"(9 + i) : "memory");
}

// One value of the cache, as it stands in the pool.
template <bool kE4m3>
__device__ float cached_value(const PoolView &pool, int64_t page, int layer, int kv, int h, int r, int d) {
    const int G = pool.n_head_kv;
    if (kE4m3) {
        const uint8_t *unit = pool.base + code_unit_index(page, layer, h, pool.n_pages, G) * kCodeUnitBytes;
        const uint32_t c =
            unit[kv * kCodeBlockBytes + r * kHeadDim + (((d >> 4) ^ (r & 7)) << 4) + (d & 15)];
        return codes_to_float4(c).x * pow2(reinterpret_cast<const int *>(unit + 2 * kCodeBlockBytes)[kv]);
    }
    const uint8_t *b = pool.base + head_block_index(page, layer, kv, h, pool.n_pages, G) * kHeadBlockBytes;
    return __half2float(
        *reinterpret_cast<const __half *>(b + r * kRowBytes + swizzled_chunk(r, d >> 3) * 16 + (d & 7) * 2));
}

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(d)
        : "l"(*reinterpret_cast<const uint64_t *>(&a)), "l"(*reinterpret_cast<const uint64_t *>(&b)),
          "l"(*reinterpret_cast<const uint64_t *>(&c)));
    return *reinterpret_cast<const float2 *>(&d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(d)
        : "l"(*reinterpret_cast<const uint64_t *>(&a)), "l"(*reinterpret_cast<const uint64_t *>(&b)));
    return *reinterpret_cast<const float2 *>(&d);
}

// The issuing thread of M tile i: S_i = q_i K^T and O_i += P_i V, block by block.  nb:
// blocks of the CTA, blocks: of the tile.  Each tile has its own issuer, since a wait or
// commit costs one about 130 cycles during which only the other's products are queued.
template <class S>
__device__ __forceinline__ void issue_products(Control *ctl, uint32_t q_addr, uint32_t k_ring, uint32_t v_ring,
                                               uint32_t tmem, int i, int nb, int blocks, DeviceError *err) {
    constexpr uint32_t qk_desc = mma_idesc(kTile, kKeys, false);
    constexpr uint32_t pv_desc = mma_idesc(kTile, kHeadDim, true);
    auto k_ready = [&](int j) {
        return wait_for(&ctl->k_full[j % S::kKSlots], (j / S::kKSlots) & 1, err);
    };
    auto v_ready = [&](int j) {
        return wait_for(&ctl->v_full[j % S::kVSlots], (j / S::kVSlots) & 1, err);
    };
    auto logits = [&](int j) {  // S_i of block j
        const uint32_t kb = k_ring + (j % S::kKSlots) * S::kKTile;
        // the low part first: the tensor cores' F32 sums are cut, not rounded, and its own
        // are 2^-11 as large
#pragma unroll
        for (int part = S::kParts - 1; part >= 0; --part) {
            const uint32_t qa = q_addr + (i * S::kParts + part) * S::kQPart;
            if (S::kCodeK) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    mma_ss_e4m3(tmem + i * kKeys, smem_desc(qa + k * 32, 16, 1024), smem_desc(kb + k * 32, 16, 1024),
                                qk_desc, part < S::kParts - 1 || k > 0);
                }
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const uint32_t step = (k >> 2) * (kTileBytes / 2) + (k & 3) * 32;
                    mma_ss(tmem + i * kKeys, smem_desc(qa + step, 16, 1024), smem_desc(kb + step, 16, 1024), qk_desc,
                           part < S::kParts - 1 || k > 0);
                }
            }
        }
        tc_commit(smem_u32(&ctl->s_full[i]));
    };
    auto weigh = [&](int j, int c) {  // O_i += P_i V of block j, the keys that p_full[i][c] stands for
        const uint32_t vb = v_ring + (j % S::kVSlots) * kTileBytes;
#pragma unroll
        for (int part = 0; part < (S::kSplit ? 2 : 1); ++part) {
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const int k = 4 * (n >> 1) + 2 * c + (n & 1);
                const uint32_t p = tmem + i * kKeys + (k >> 1) * 32 + part * 16 + (k & 1) * 8;
                mma_ts(tmem + 256 + i * kHeadDim, p, smem_desc(vb + k * 2048, kTileBytes / 2, 1024), pv_desc,
                       (S::kSplit ? j % kDrainBlocks : j) > 0 || part > 0 || c > 0 || n > 0);
            }
        }
    };
    // The issuers take turns, so that a tile's products stand in line as a whole: mixed,
    // both tiles would get theirs late, and at the same time, and their softmaxes would
    // then compete for the exponentials.
    auto turn = [&](int round) { return wait_for(&ctl->turn[i], round & 1, err); };
    auto pass = [&]() { mbar_arrive(smem_u32(&ctl->turn[i ^ 1])); };
    bool ok = (blocks == 0 || (wait_for(&ctl->q_full, 0, err) && k_ready(0))) && turn(0);
    if (ok && blocks > 0) {
        logits(0);
        tc_commit(smem_u32(&ctl->k_empty[0]));
    }
    pass();
    for (int j = 0; ok && j < nb; ++j) {
        if (j >= blocks) {
            // a block that only the other tile takes: its buffers are let go at once (the
            // other issuer may wait for them in its turn)
            ok = k_ready(j);
            if (ok) {
                mbar_arrive(smem_u32(&ctl->k_empty[j % S::kKSlots]));
                ok = v_ready(j);
            }
            if (ok) {
                mbar_arrive(smem_u32(&ctl->v_empty[j % S::kVSlots]));
                ok = turn(j + 1);
            }
            if (ok) {
                pass();
            }
            continue;
        }
        const bool more = j + 1 < blocks;
        ok = v_ready(j);
        if (S::kEarly) {
            ok = ok && wait_for(&ctl->p_full[i][0], j & 1, err);
            if (!ok) {
                break;
            }
            tc_fence_after();
            weigh(j, 0);
        }
        ok = ok && (S::kKSlots == 1 || !more || k_ready(j + 1)) && wait_for(&ctl->p_full[i][1], j & 1, err) && turn(j + 1);
        if (!ok) {
            break;
        }
        tc_fence_after();
        if (!S::kEarly) {
            weigh(j, 0);
        }
        weigh(j, 1);
        if (more) {
            ok = S::kKSlots > 1 || k_ready(j + 1);
            if (!ok) {
                break;
            }
            logits(j + 1);
        } else {
            tc_commit(smem_u32(&ctl->o_full[i]));
        }
        pass();
        if (more) {
            tc_commit(smem_u32(&ctl->k_empty[(j + 1) % S::kKSlots]));
        }
        tc_commit(smem_u32(&ctl->v_empty[j % S::kVSlots]));
    }
    if (!ok) {
        // products in flight end before the memory they use is given up
        tc_commit(smem_u32(&ctl->drained[i]));
        mbar_wait_bounded(smem_u32(&ctl->drained[i]), 0);
    }
}

template <typename T, bool kE4m3>
__global__ void __launch_bounds__(kThreads, 1)
    window_kernel(PoolView pool, const WindowTile *__restrict__ tiles, const int32_t *__restrict__ pages, int layer,
                  const T *__restrict__ q, int64_t q_stride, T *__restrict__ out, int64_t out_stride,
                  float *__restrict__ work, float scale_log2, DeviceError *err) {
    using S = Shape<T, kE4m3>;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t q_smem = smem_u32(smem);
    const uint32_t k_ring = q_smem + S::kQBytes;
    const uint32_t v_ring = k_ring + S::kKSlots * S::kKTile;
    Control *ctl = reinterpret_cast<Control *>(smem + S::kControl);
    BlockScale *scales = reinterpret_cast<BlockScale *>(ctl + 1);
    const int G = pool.n_head_kv;
    // The heads of a tile stand together, so that CTAs start in the order of the tiles,
    // longest first: 8100 F32 tokens 1033 us, BF16 615, 8 ragged windows F32 461, BF16 279;
    // with all tiles of a head, then the next head's, 1214, 630, 488 and 273
    const int h = blockIdx.x % G;
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    if (warp == kIssuer) {
        tmem_alloc(smem_u32(&ctl->tmem), 512);
    }
    if (threadIdx.x == 0) {
        mbar_init(smem_u32(&ctl->q_full), kSoftmaxThreads);
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&ctl->s_full[i]), 1);
            mbar_init(smem_u32(&ctl->p_full[i][0]), kTileThreads);
            mbar_init(smem_u32(&ctl->p_full[i][1]), kTileThreads);
            mbar_init(smem_u32(&ctl->o_full[i]), 1);
            mbar_init(smem_u32(&ctl->drained[i]), 1);
        }
        for (int i = 0; i < S::kKSlots; ++i) {
            mbar_init(smem_u32(&ctl->k_full[i]), S::kCodeK ? 2 : kConvertThreads + 1);
            mbar_init(smem_u32(&ctl->k_empty[i]), 2);
        }
        for (int i = 0; i < S::kVSlots; ++i) {
            mbar_init(smem_u32(&ctl->v_full[i]), kConvertThreads);
            mbar_init(smem_u32(&ctl->v_empty[i]), 2);
        }
        mbar_init(smem_u32(&ctl->turn[0]), 1);
        mbar_init(smem_u32(&ctl->turn[1]), 1);
        mbar_arrive(smem_u32(&ctl->turn[0]));
        ctl->odd_v = 0;
        fence_barrier_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctl->tmem;
    // set up while the kernel before this one ended; its writes from here on
    pdl_wait();
    pdl_trigger();
    const WindowTile t = tiles[blockIdx.x / G];
    const int n_tiles = t.tokens > kTileTokens ? 2 : 1;
    // blocks of each M tile: up to the last key that its last token sees
    const int key_end0 = t.pos0 + min(t.tokens, kTileTokens) - t.key0;
    const int nb0 = min(t.blocks, max(0, (key_end0 + kKeys - 1) / kKeys));
    const int nb1 = n_tiles == 2 ? t.blocks : 0;
    const int nb = max(nb0, nb1);


    // The slot's pages from the CTA's first key on.  Past its last one that one is
    // read again: K there is masked, V zeroed.
    const int32_t *list = pages + t.page_off + t.key0 / kPageTokens;
    const int last_page = (t.pos0 + t.tokens - 1 - t.key0) / kPageTokens;
    const int last_key = t.pos0 + t.tokens - 1 - t.key0;
    const int64_t page_stride = static_cast<int64_t>(G) * cache_unit_bytes(kE4m3 ? kCacheE4m3 : kCacheF16);
    const uint8_t *head_base = pool.base + static_cast<int64_t>(layer) * pool.n_pages * page_stride +
                               h * (kE4m3 ? kCodeUnitBytes : kHeadBlockBytes);
    int bad = -1;  // index of a page id outside the pool
    auto page_at = [&](int index) {
        int page = list[min(index, last_page)];
        if (page >= pool.n_pages || page < 0) {
            bad = index;
            page = 0;
        }
        return page;
    };

    if (warp < kSoftmaxThreads / 32) {
        // ------------------------------------------------------------ softmax
        take_registers<kSoftmaxRegs>();
        const int i = warp >> 3;                      // M tile
        const int half = (warp >> 2) & 1;             // of a block's keys, and of o's dims
        const int row = (warp & 3) * 32 + lane;       // = 4 token + head
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t s_col = tmem + lanes + i * kKeys + half * 64;
        const uint32_t o_col = tmem + lanes + 256 + i * kHeadDim + half * 64;
        // q: sixteen lanes hold a row, 8 dims each; rows past the last token are zeros
#pragma unroll 2
        for (int it = 0; it < 8; ++it) {
            const int idx = it * kTileThreads + half * kTile + row;
            const int r = idx >> 4;
            const int c = idx & 15;
            const int tok = i * kTileTokens + (r >> 2);
            float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (tok < t.tokens) {
                load8(q + (static_cast<int64_t>(t.row0) + tok) * q_stride + (kGqa * h + (r & 3)) * kHeadDim + c * 8, x);
            }
            const uint32_t part0 = q_smem + i * S::kParts * S::kQPart;
            if (S::kCodeK) {
                float amax = 0.f;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    amax = fmaxf(amax, finite_abs(x[k]));
                }
#pragma unroll
                for (int off = 8; off > 0; off >>= 1) {
                    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
                }
                const int e = max(block_exponent(amax), kQExpMin);
                if (c == 0) {
                    ctl->rows[i].q_exp[r] = e;
                }
                const float inv = pow2(-e);
                uint32_t hi[2], lo[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float4 y = make_float4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]);
                    hi[k] = to_codes4(y, inv);
                    const float4 f = codes_to_float4(hi[k]);
                    lo[k] = to_codes4(make_float4(fmaf(y.x, inv, -f.x), fmaf(y.y, inv, -f.y), fmaf(y.z, inv, -f.z),
                                                  fmaf(y.w, inv, -f.w)),
                                      1.f);
                }
                const uint32_t at = part0 + r * kHeadDim + (((c >> 1) ^ (r & 7)) << 4) + (c & 1) * 8;
                st_shared8(at, hi[0], hi[1]);
                st_shared8(at + S::kQPart, lo[0], lo[1]);
            } else {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    hi[k] = half2_bits(x[2 * k], x[2 * k + 1]);
                    const float2 f = half2_floats(hi[k]);
                    lo[k] = half2_bits(__fsub_rn(x[2 * k], f.x), __fsub_rn(x[2 * k + 1], f.y));
                }
                const uint32_t at = part0 + tile_offset(kTile, r, c);
                st_shared16(at, hi[0], hi[1], hi[2], hi[3]);
                if (S::kSplit) {
                    st_shared16(at + S::kQPart, lo[0], lo[1], lo[2], lo[3]);
                }
            }
        }
        fence_proxy_async_smem();
        mbar_arrive(smem_u32(&ctl->q_full));
        float q_scale = 1.f;
        if (S::kCodeK) {
            tile_barrier(i);  // q_exp of the tile's rows
            q_scale = pow2(ctl->rows[i].q_exp[row]);
            tile_barrier(i);  // before `half` takes its place
        }

        const int my_tok = i * kTileTokens + (row >> 2);
        const int my_last = t.pos0 + min(my_tok, t.tokens - 1) - t.key0;  // last key this row sees
        const int first_last = t.pos0 + i * kTileTokens - t.key0;         // and the tile's first row
        const int blocks = i == 0 ? nb0 : nb1;
        float m = -INFINITY, l = 0.f;
        // What a page's products are multiplied by: with K's exponents up to 120 and those of q,
        // |q| <= 65504, up to 8, a finite float.
        auto logit_scale = [&](const PageScale &page) {
            return S::kCodeK ? page.k * q_scale : page.k;
        };
        const bool live = my_tok < t.tokens;
        // the token's four rows, from this lane's dims on
        const int my_dim = 64 * half + 4 * (lane & 3);
        T *dst = out + (static_cast<int64_t>(t.row0) + my_tok) * out_stride + kGqa * h * kHeadDim + my_dim;
        float *part = work + (static_cast<int64_t>(t.part) * G + h) * kWindowPartFloats;
        float *part_rows = part + (i * kTile + (row & ~3)) * kHeadDim + my_dim;
        // F32 tensors: where o is added up, and what that sum has to be multiplied by
        float *sums = t.part >= 0 ? part_rows : reinterpret_cast<float *>(dst);
        const bool keeps = t.part >= 0 || live;
        float kept = 0.f;
        int j = 0;
        for (; j < blocks; ++j) {
            if (!__all_sync(0xffffffffu, wait_for(&ctl->s_full[i], j & 1, err))) {
                break;
            }
            tc_fence_after();
            const BlockScale &b = scales[j % S::kScaleSlots];
            const bool masked = j * kKeys + 64 * half + 63 > first_last;
            const int lim = my_last - j * kKeys - 64 * half;  // columns 0 .. lim of this half are seen
            float mx = -INFINITY;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float s[32];
                tmem_load32(s_col + 32 * c, s);
                if (masked) {
#pragma unroll
                    for (int k = 0; k < 32; ++k) {
                        s[k] = 32 * c + k <= lim ? s[k] : -INFINITY;
                    }
                }
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    float a = s[16 * p], d = s[16 * p + 1];
#pragma unroll
                    for (int k = 2; k < 14; k += 4) {
                        a = max3(a, s[16 * p + k], s[16 * p + k + 1]);
                        d = max3(d, s[16 * p + k + 2], s[16 * p + k + 3]);
                    }
                    a = max3(a, s[16 * p + 14], s[16 * p + 15]);
                    const PageScale page = b.page[4 * half + 2 * c + p];
                    mx = fmaxf(mx, fmaf(fmaxf(a, d), logit_scale(page), kE4m3 ? page.v_exp : 0.f));
                }
            }
            // the row's bound over both halves
            ctl->rows[i].half[half][row] = mx;
            pair_barrier(warp);
            mx = fmaxf(mx, ctl->rows[i].half[half ^ 1][row]);
            const bool drain = S::kSplit && j > 0 && j % kDrainBlocks == 0;
            if (drain) {
                // brought to the sums' units, where those are not too far (2^60 leaves a
                // sum of 2^9 weights of 2^15 and V of 2^16 below 2^100), for an addition in
                // L2 that nothing waits for
                const bool first = j == kDrainBlocks;
                const bool in_place = !first && __all_sync(0xffffffffu, kept >= 0x1p-60f);
                const float4 scale = of_rows(in_place ? 1.f / kept : kept, lane);
#pragma unroll 1
                for (int c = 0; c < 64; c += 16) {
                    float o[16];
                    tmem_load16(o_col + c, o);
                    four_rows(o, lane);
                    if (keeps && in_place) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                o[4 * r + k] *= row_of(scale, r);
                            }
                            add_at(sums + r * kHeadDim + c, o + 4 * r);
                        }
                    } else if (keeps) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            if (!first) {
                                plus4(o + 4 * r, load_at(sums + r * kHeadDim + c), row_of(scale, r));
                            }
                            store4(sums + r * kHeadDim + c, o + 4 * r);
                        }
                    }
                }
                kept = in_place ? kept : 1.f;
            }
            // the bound moves (o has to follow) only when it must
            if (__any_sync(0xffffffffu, mx > m + kSlack)) {
                const float m_new = fmaxf(m, mx);
                const float corr = (m_new == -INFINITY ? 1.f : exp2_fast(m - m_new));
                if (kE4m3) {
                    // in two steps: where V's exponent makes the bound jump, corr may
                    // underflow though the keys so far weigh
                    const float h = m_new == -INFINITY ? 1.f : exp2_fast(0.5f * (m - m_new));
                    l = l * h * h;
                } else {
                    l *= corr;
                }
                m = m_new;
                kept *= corr;
                if (j > 0 && !drain) {
#pragma unroll 1
                    for (int c = 0; c < 64; c += 16) {
                        float o[16];
                        tmem_load16(o_col + c, o);
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            o[k] *= corr;
                        }
                        tmem_store16(o_col + c, reinterpret_cast<const uint32_t (&)[16]>(o));
                    }
                }
            }
            const float bound = m == -INFINITY ? 0.f : m;
            const bool far = kE4m3 && b.far != 0;
            const bool huge = __any_sync(0xffffffffu, fabsf(bound) > kHuge);  // of a row of the warp
            if (far || huge) {
#pragma unroll 1
                for (int p = 0; p < 4; ++p) {
                    const PageScale page = b.page[4 * half + p];
                    const float sc = logit_scale(page);
                    float s[16];
                    tmem_load16(s_col + 16 * p, s);
                    float r = -INFINITY;
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        s[k] = 16 * p + k <= lim ? s[k] : -INFINITY;
                        r = fmaxf(r, s[k] * sc);
                    }
                    if (far) {
                        // V exponents far apart (`back` is 0): the page's terms of the sum by
                        // its own largest logit, and from there to the sum's units in two
                        // steps that do not underflow
                        const float top = r == -INFINITY ? 0.f : r;
                        float terms = 0.f;
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            terms += exp2_fast(__fmul_rn(s[k], sc) - top);
                        }
                        const float h = exp2_fast(0.5f * (r - bound));
                        l = fmaf(terms * h, h, l);
                    }
                    if (huge) {
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            s[k] = fmaf(s[k], sc, kE4m3 ? page.v_exp : 0.f) - bound;
                        }
                        tmem_store16(s_col + 16 * p, reinterpret_cast<const uint32_t (&)[16]>(s));
                    }
                }
                tmem_store_wait();
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float s[32];
                tmem_load32(s_col + 32 * c, s);
                if (masked) {
#pragma unroll
                    for (int k = 0; k < 32; ++k) {
                        s[k] = 32 * c + k <= lim ? s[k] : -INFINITY;
                    }
                }
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const PageScale page = b.page[4 * half + 2 * c + p];
                    const float sc = huge ? 1.f : logit_scale(page);
                    const float sh = huge ? static_cast<float>(kShift) : page.shift - bound;
                    float2 *x = reinterpret_cast<float2 *>(s + 16 * p);
                    const float2 scale = make_float2(sc, sc), off = make_float2(sh, sh);
                    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const float2 e = fma2(x[k], scale, off);
                        x[k] = make_float2(exp2_fast(e.x), exp2_fast(e.y));
                        sum = add2(sum, x[k]);
                    }
                    if (!kE4m3) {
                        l += sum.x + sum.y;  // with the 2^kShift of o
                    } else {
                        l = fmaf(sum.x + sum.y, page.back, l);
                    }
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        if (S::kSplit && kE4m3) {
                            // cut, not rounded, so that the low part does not wait for
                            // the high one's conversion: 22 bits all the same (two more
                            // registers, which the form for F16 pages does not have)
                            const float2 f = make_float2(__uint_as_float(__float_as_uint(x[k].x) & 0xffffe000u),
                                                         __uint_as_float(__float_as_uint(x[k].y) & 0xffffe000u));
                            const float2 r = fma2(f, make_float2(-1.f, -1.f), x[k]);
                            hi[8 * p + k] = half2_bits(f.x, f.y);
                            lo[8 * p + k] = half2_bits(r.x, r.y);
                        } else {
                            hi[8 * p + k] = half2_bits(x[k].x, x[k].y);
                            if (S::kSplit) {
                                const float2 f = half2_floats(hi[8 * p + k]);
                                lo[8 * p + k] = half2_bits(x[k].x - f.x, x[k].y - f.y);
                            }
                        }
                    }
                }
                // in place of the logits: 16 columns of hi, 16 of lo per 32 keys
                tmem_store16(s_col + 32 * c, hi);
                if (S::kSplit) {
                    tmem_store16(s_col + 32 * c + 16, lo);
                }
                if (S::kEarly || c == 1) {
                    tmem_store_wait();
                    tc_fence_before();
                    mbar_arrive(smem_u32(&ctl->p_full[i][c]));
                }
            }
        }
        // The two warps of a row pair find out on their own that a wait ran out, at different
        // blocks perhaps.  One that did goes to the barriers that are left, so that its
        // partner meets it at each: one per block and one at the end.
        bool ok = j == blocks;
        for (; j < blocks; ++j) {
            pair_barrier(warp);
        }
        if (ok && blocks > 0) {
            ok = __all_sync(0xffffffffu, wait_for(&ctl->o_full[i], 0, err));
        }
        // the row's sum over both halves (bounds are the same)
        if (blocks > 0) {
            ctl->rows[i].half[half][row] = l;
            pair_barrier(warp);
            l += ctl->rows[i].half[half ^ 1][row];
        }
        if (ok) {
            tc_fence_after();
            const uint32_t odd = *reinterpret_cast<volatile uint32_t *>(&ctl->odd_v);
            // F16 cache: o and l carry 2^kShift, a part's o is not normalised.  8-bit cache:
            // o carries it, and a part's l and o are brought to l in [1, 2) by a power of two
            // that m takes up, which is then the size of a logit again; both times 2^-12, so
            // that no join of up to 2^11 parts overflows.
            float own = t.part < 0 ? 1.f / l : 1.f;
            if (kE4m3 && t.part >= 0) {
                const int e = min(max(static_cast<int>((__float_as_uint(l) >> 23) & 255u) - 127, -126), 114);
                own = pow2(-e - 12);
                l *= own;
                m += static_cast<float>(e);
            }
            constexpr float kUnit = kE4m3 ? 1.f / (1 << kShift) : 1.f;
            const float4 f = of_rows(own, lane);
            const float4 scale = of_rows(kept, lane);
#pragma unroll 1
            for (int c = 0; c < 64; c += 16) {
                float o[16];
                if (blocks > 0) {
                    tmem_load16(o_col + c, o);
                }
                four_rows(o, lane);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (S::kSplit && blocks > kDrainBlocks && keeps) {
                        plus4(o + 4 * r, load_at(sums + r * kHeadDim + c), row_of(scale, r));
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        o[4 * r + k] = blocks > 0 ? o[4 * r + k] * kUnit * row_of(f, r) : 0.f;
                    }
                }
                if (odd != 0 && live) {
                    const int keys = min(my_last + 1, t.blocks * kKeys);
                    for (int key = 0; key < keys; ++key) {
                        if ((odd >> (key / kKeys & 31) & 1u) == 0) {
                            key += kKeys - 1;
                            continue;
                        }
                        const int page = page_at(key / kPageTokens);
#pragma unroll 1
                        for (int k = 0; k < 4; ++k) {
                            const float x = cached_value<kE4m3>(pool, page, layer, 1, h, key & 15, my_dim + c + k);
                            if (!(fabsf(x) <= 3.402823466e38f)) {
#pragma unroll
                                for (int z = 0; z < 16; ++z) {
                                    o[z] += (z & 3) == k ? x : 0.f;
                                }
                            }
                        }
                    }
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (t.part >= 0) {
                        store4(part_rows + r * kHeadDim + c, o + 4 * r);
                    } else if (live) {
                        store4(dst + r * kHeadDim + c, o + 4 * r);
                    }
                }
            }
            if (t.part >= 0 && half == 0) {
                float2 *ml = reinterpret_cast<float2 *>(part + kWindowTokens * kGqa * kHeadDim);
                ml[i * kTile + row] = make_float2(m, l);
            }
            tc_fence_before();
        }
    } else {
        give_registers<kOtherRegs>();
        if (warp < kScaleWarp) {
            // -------------------------------------------------------- converters
            const int tid = threadIdx.x - kSoftmaxThreads;
            // A half tile is 1024 (F16: a quarter, 512 x 2) 16-byte pieces: 8 bits, 16 dims of a
            // row; F16, 8 dims.  Steps of 1024 pieces, K (where it is converted) then V of
            // each block; the pieces of the next step are in registers: its loads go out
            // when the step before it is stored.
            // Eight consecutive threads store to eight different bank groups: 8 bits, dims
            // 0-63 or 64-127 of two neighbouring rows (an even and an odd row's swizzles
            // interleave); F16, half a row.
            constexpr int kTileSteps = kE4m3 ? 1 : 2;
            constexpr int kSteps = (S::kCodeK ? 1 : 2) * kTileSteps;
            constexpr int kAhead = 1;
            constexpr int kPieces = 1024;
            constexpr int kEach = (kPieces + kConvertThreads - 1) / kConvertThreads;
            static_assert(kConvertThreads % 16 == 0, "a thread keeps its place in the row");
            const int c = kE4m3 ? ((tid >> 3) & 1) * 4 + (tid & 3) : tid & 15;  // piece of the row
            const int row0 = kE4m3 ? 2 * (tid >> 4) + ((tid >> 2) & 1) : tid >> 4;
            constexpr int kRowStep = (kE4m3 ? 2 : 1) * kConvertThreads / 16;
            const int64_t v_off = kE4m3 ? kCodeBlockBytes : static_cast<int64_t>(G) * kHeadBlockBytes;
            auto step_is_v = [](int step) { return S::kCodeK || step >= kTileSteps; };
            uint4 raw[kAhead][kEach];
            auto fetch = [&](int j, int step, uint4 (&to)[kEach]) {
                const uint8_t *from = head_base + (step_is_v(step) ? v_off : 0);
                const int first = j * kBlockPages + (kE4m3 ? 0 : (step & 1) * 4);
                int page[kEach];
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    page[i] = page_at(first + ((row0 + i * kRowStep) >> 4));
                }
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    const int row = (row0 + i * kRowStep) & 15;
                    to[i] = *reinterpret_cast<const uint4 *>(from + page[i] * page_stride +
                                                             row * (kE4m3 ? kHeadDim : kRowBytes) +
                                                             ((c ^ (row & 7)) << 4));
                }
            };
            auto put = [&](int j, int step, const uint4 (&from)[kEach], uint32_t buf) {
                const bool is_v = step_is_v(step);
                const bool tail = is_v && j * kKeys + kKeys - 1 > last_key;
                bool odd = false;
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    const int row = (kE4m3 ? 0 : 64 * (step & 1)) + row0 + i * kRowStep;
                    if (i == kEach - 1 && tid + i * kConvertThreads >= kPieces) {
                        break;
                    }
                    uint32_t w[4] = {from[i].x, from[i].y, from[i].z, from[i].w};
                    // rows past the last key hold whatever the page had before
                    if (tail && j * kKeys + row > last_key) {
                        w[0] = w[1] = w[2] = w[3] = 0;
                    }
                    uint32_t x[kE4m3 ? 8 : 4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if (kE4m3) {
                            x[2 * k] = codes_to_half2(w[k]);
                            x[2 * k + 1] = codes_to_half2_hi(w[k]);
                        } else {
                            x[k] = w[k];
                        }
                    }
                    if (is_v) {
                        // a sum that is not finite: look at each (an F16 sum may overflow)
                        uint32_t sum = x[0];
#pragma unroll
                        for (int k = 1; k < (kE4m3 ? 8 : 4); ++k) {
                            sum = half2_sum(sum, x[k]);
                        }
                        if ((((sum & 0x7c007c00u) + 0x04000400u) & 0x80008000u) != 0) {
#pragma unroll
                            for (int k = 0; k < (kE4m3 ? 8 : 4); ++k) {
                                const uint32_t out = ((x[k] & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
                                odd = odd || out != 0;
                                x[k] &= ~((out >> 15) * 0xffffu);
                            }
                        }
                    }
                    if (kE4m3) {
                        st_shared16(buf + tile_offset(kKeys, row, 2 * c), x[0], x[1], x[2], x[3]);
                        st_shared16(buf + tile_offset(kKeys, row, 2 * c + 1), x[kE4m3 ? 4 : 0], x[kE4m3 ? 5 : 0],
                                    x[kE4m3 ? 6 : 0], x[kE4m3 ? 7 : 0]);
                    } else {
                        st_shared16(buf + tile_offset(kKeys, row, c), x[0], x[1], x[2], x[3]);
                    }
                }
                if (odd) {
                    atomicOr(&ctl->odd_v, 1u << (j & 31));
                }
            };
            // steps in one line, step s of block j being j * kSteps + s
            const int all = nb * kSteps;
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                if (a < all) {
                    fetch(a / kSteps, a % kSteps, raw[a]);
                }
            }
            bool ok = true;
            for (int first = 0; ok && first < all; first += kAhead) {
#pragma unroll
                for (int a = 0; a < kAhead; ++a) {
                    const int at = first + a;
                    if (at >= all) {
                        break;
                    }
                    const int j = at / kSteps;
                    const int step = at % kSteps;
                    const bool is_v = step_is_v(step);
                    const int slot = is_v ? j % S::kVSlots : j % S::kKSlots;
                    if (step % kTileSteps == 0) {
                        const int n = is_v ? S::kVSlots : S::kKSlots;
                        if (j >= n && !wait_for(is_v ? &ctl->v_empty[slot] : &ctl->k_empty[slot], (j / n - 1) & 1, err)) {
                            ok = false;
                            break;
                        }
                    }
                    put(j, step, raw[a], is_v ? v_ring + slot * kTileBytes : k_ring + slot * S::kKTile);
                    if (step % kTileSteps == kTileSteps - 1) {
                        fence_proxy_async_smem();
                        mbar_arrive(smem_u32(is_v ? &ctl->v_full[slot] : &ctl->k_full[slot]));
                    }
                    if (at + kAhead < all) {
                        fetch((at + kAhead) / kSteps, (at + kAhead) % kSteps, raw[a]);
                    }
                }
            }
        } else if (warp == kScaleWarp) {
            // ------------------------------------------- exponents, and K's codes
            int e = INT32_MIN;  // the largest V exponent so far
            bool ok = true;
            for (int j = 0; ok && j < nb; ++j) {
                const int slot = j % S::kKSlots;
                const uint32_t bar = smem_u32(&ctl->k_full[slot]);
                const int index = j * kBlockPages + (lane & 7);
                const bool there = index <= last_page;
                const int64_t page = page_at(index);
                const uint8_t *unit = head_base + page * page_stride;
                int2 exps = make_int2(0, 0);
                if (kE4m3) {
                    exps = *reinterpret_cast<const int2 *>(unit + 2 * kCodeBlockBytes);
                }
                if (j >= S::kKSlots) {
                    ok = __all_sync(0xffffffffu, wait_for(&ctl->k_empty[slot], (j / S::kKSlots - 1) & 1, err));
                    if (!ok) {
                        break;
                    }
                }
                if (S::kCodeK) {
                    // the copies go out before the exponents are looked at
                    if (lane == 0) {
                        mbar_arrive_expect_tx(bar, kCodeTileBytes);
                    }
                    __syncwarp();
                    if (lane < kBlockPages) {
                        bulk_load(k_ring + slot * S::kKTile + lane * kCodeBlockBytes, unit, kCodeBlockBytes, bar,
                                  keep_policy());
                    }
                }
                int top = there ? exps.y : INT32_MIN;
#pragma unroll
                for (int off = 4; off > 0; off >>= 1) {
                    top = max(top, __shfl_xor_sync(0xffffffffu, top, off));
                }
                e = max(e, top);
                const int e_v = there ? exps.y : 0;
                const bool far = __any_sync(0xffffffffu, there && e_v < e - kFar);
                BlockScale &b = scales[j % S::kScaleSlots];
                if (lane < kBlockPages) {
                    b.page[lane] = {scale_log2 * pow2(exps.x), static_cast<float>(e_v), static_cast<float>(kShift + e_v),
                                    far ? 0.f : ldexpf(1.f, -(kShift + e_v))};
                }
                if (lane == 0) {
                    b.far = far ? 1 : 0;
                }
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(bar);
                }
            }
            if (S::kCodeK) {
                // copies that no product waited for end before the CTA does
                for (int j = max(0, nb - S::kKSlots); j < nb; ++j) {
                    mbar_wait_bounded(smem_u32(&ctl->k_full[j % S::kKSlots]), (j / S::kKSlots) & 1);
                }
            }
        } else if (lane == 0) {
            // ---------------------------------------------------------- products
            const int i = warp - kIssuer;
            issue_products<S>(ctl, q_smem, k_ring, v_ring, tmem, i, nb, i == 0 ? nb0 : nb1, err);
        }
    }
    if (bad >= 0) {
        record(err, kErrBadIndex, list[min(bad, last_page)], bad);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kIssuer) {
        __syncwarp();
        tmem_free(tmem, 512);
    }
}

// Joins the parts of a split tile: one warp a row, in part order.
template <typename T>
__global__ void __launch_bounds__(256)
    window_combine_kernel(const WindowMerge *__restrict__ merges, int G, const float *__restrict__ work,
                          T *__restrict__ out, int64_t out_stride) {
    pdl_wait();
    pdl_trigger();
    const WindowMerge g = merges[blockIdx.x];
    const int h = blockIdx.y;
    const int row = blockIdx.z * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (row >= g.tokens * kGqa) {
        return;
    }
    auto part = [&](int p) { return work + (static_cast<int64_t>(g.part0 + p) * G + h) * kWindowPartFloats; };
    auto stats = [&](int p) {
        return reinterpret_cast<const float2 *>(part(p) + kWindowTokens * kGqa * kHeadDim)[row];
    };
    float m = -INFINITY;
    for (int p = 0; p < g.parts; ++p) {
        m = fmaxf(m, stats(p).x);
    }
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
    for (int p = 0; p < g.parts; ++p) {
        const float2 ml = stats(p);
        const float4 o = reinterpret_cast<const float4 *>(part(p) + row * kHeadDim)[lane];
        if (ml.x == -INFINITY && ml.y == 0.f) {
            continue;  // a part whose keys this row does not see
        }
        const float w = exp2f(ml.x - m);
        l += w * ml.y;
        acc.x += w * o.x;
        acc.y += w * o.y;
        acc.z += w * o.z;
        acc.w += w * o.w;
    }
    const float x[4] = {acc.x / l, acc.y / l, acc.z / l, acc.w / l};
    store4(out + (static_cast<int64_t>(g.row0) + (row >> 2)) * out_stride + (kGqa * h + (row & 3)) * kHeadDim + 4 * lane, x);
}

template <typename T, bool kE4m3>
void launch_window_t(const PoolView &pool, const WindowArgs &a, DeviceError *err, cudaStream_t stream) {
    static bool configured[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        cudaFuncSetAttribute(window_kernel<T, kE4m3>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<T, kE4m3>::kSmem);
        if (dev >= 0 && dev < 64) {
            configured[dev] = true;
        }
    }
    const unsigned G = static_cast<unsigned>(pool.n_head_kv);
    T *out = static_cast<T *>(a.out);
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(a.n_tiles) * G);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Shape<T, kE4m3>::kSmem;
    cfg.stream = stream;
    cfg.attrs = &attr;
    // A launch of one wave is set up while the kernel before it runs (37 tokens behind
    // 770: 16.7 us, 18.6 without); of one of several waves the first CTAs would wait in the
    // places of the last (8100 tokens F32 1033 us, 1049 so; BF16 within 1%).
    cfg.numAttrs = a.one_wave ? 1 : 0;
    cudaLaunchKernelEx(&cfg, window_kernel<T, kE4m3>, pool, a.tiles, a.pages, a.layer, static_cast<const T *>(a.q),
                       a.q_stride, out, a.out_stride, a.work, a.scale_log2, err);
    if (a.n_merges > 0) {
        cfg.gridDim = dim3(static_cast<unsigned>(a.n_merges), G, kWindowTokens * kGqa / 8);
        cfg.blockDim = dim3(256);
        cfg.dynamicSmemBytes = 0;
        cfg.numAttrs = 1;
        cudaLaunchKernelEx(&cfg, window_combine_kernel<T>, a.merges, static_cast<int>(G),
                           static_cast<const float *>(a.work), out, a.out_stride);
    }
}

template <typename T>
void launch_window_f(const PoolView &pool, const WindowArgs &a, DeviceError *err, cudaStream_t stream) {
    if (pool.format == kCacheE4m3) {
        launch_window_t<T, true>(pool, a, err, stream);
    } else {
        launch_window_t<T, false>(pool, a, err, stream);
    }
}

}  // namespace

void launch_window(const PoolView &pool, const WindowArgs &args, DeviceError *err, cudaStream_t stream) {
    if (args.dtype == kDtypeF32) {
        launch_window_f<float>(pool, args, err, stream);
    } else if (args.dtype == kDtypeF16) {
        launch_window_f<__half>(pool, args, err, stream);
    } else {
        launch_window_f<__nv_bfloat16>(pool, args, err, stream);
    }
}

}  // namespace hkv
