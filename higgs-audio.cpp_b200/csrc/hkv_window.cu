// hkv_window.cu -- attention of several new tokens per slot over the paged cache
// (prompts, refreshed windows): row i of a slot sees rows [0, used + i].
//
//   s_t = (q . c_t) 2^eK scale log2(e),  w_t = 2^(s_t - m),
//   o   = sum_t w_t 2^(eV - E) c_t,      out = o 2^E / sum_t w_t
//
// with codes c (F16 values in an F16 cache: eK = eV = 0), m a running bound of
// the logits and E the largest eV so far; one pass over the keys.
//
// One CTA takes up to 64 tokens x the 4 query heads of a KV head, as two M = 128
// tiles (row = 4 token + head), so that a key is read and converted once for 256
// rows, and a run of 128-key blocks.  Both products run on the tensor cores
// (tcgen05, F32 accumulators in TMEM); codes are exact in F16, so K and V enter
// without error.
//   warps 0-3, 4-7  softmax of M tile 0 / 1, a thread a row: S from TMEM, the
//                   weights back into S's columns as the next product's A operand
//   warps 8-10      loaders: 16-byte pieces of the pages to F16 operand tiles,
//                   through a ring of 32 KiB buffers (K and V tiles in turn)
//   warp 11         one thread issues every product; while one tile's softmax
//                   runs, the other tile's products do
// F32 tensors: q and the weights in two F16 parts each, hi + lo, which keeps 22
// bits and doubles the products.  F16 and BF16 tensors: one part.
//
// The rescaling of o when the bound m moves is put off until a row passes it by
// 2^kSlack (weights up to 2^kSlack then enter the product); o is rescaled in TMEM
// by the softmax warps, rarely after the first blocks.
//
// Non-finite V values are zeroed in the operand tiles, since 0 * inf would reach
// rows that do not see them; a CTA that met one adds them to the rows that do see
// them at its end.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

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

constexpr int kKeys = 128;              // keys of a block
constexpr int kBlockPages = kKeys / kPageTokens;
constexpr int kTile = 128;              // rows of an M tile: 32 tokens x 4 heads
constexpr int kTileTokens = kTile / kGqa;
constexpr int kTileBytes = 128 * 128 * 2;
constexpr int kSoftmaxThreads = 256;
constexpr int kLoaderThreads = 96;
// Twelve warps: 168 registers a thread, which hold a row of 128 logits.
constexpr int kThreads = kSoftmaxThreads + kLoaderThreads + 32;
constexpr int kIssuer = kThreads / 32 - 1;
constexpr int kScaleSlots = 4;          // blocks whose exponents are kept
constexpr float kSlack = 8.f;
constexpr int kShift = 7;               // weights enter 2^7 larger: at most 2^15 in F16
constexpr int kNoPage = INT32_MIN;      // exponent of V where a block has no page
constexpr int kFar = 60;                // V exponents this far below E take the slow form

template <typename T>
struct Shape {
    static constexpr bool kSplit = sizeof(T) == 4;
    static constexpr int kParts = kSplit ? 2 : 1;  // F16 parts of q and of the weights
    static constexpr int kRing = kSplit ? 3 : 5;   // operand tiles beside q in 224 KiB
    static constexpr int kQBytes = 2 * kParts * kTileBytes;
    static constexpr int kSmem = kQBytes + kRing * kTileBytes + 1024;
};

struct Control {
    uint64_t q_full, s_full[2], p_full[2], o_full[2], kv_full[5], kv_empty[5];
    uint64_t drained;                           // after a wait that ran out: no product in flight
    uint32_t tmem;
    int odd_v;                                  // a V value that is not finite was met
    float k_scale[kScaleSlots][kBlockPages];    // scale * log2(e) * 2^eK
    int v_exp[kScaleSlots][kBlockPages];
};
static_assert(sizeof(Control) <= 1024, "the control block has 1 KiB");

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

// A wait of one role.  One that runs out is recorded and ends its role; the waits
// that depend on it run out in turn, and the CTA leaves.
__device__ __forceinline__ bool wait_for(uint64_t *bar, uint32_t parity, DeviceError *err) {
    if (mbar_wait_bounded(smem_u32(bar), parity)) {
        return true;
    }
    record(err, kErrTimeout, static_cast<int>(blockIdx.x), static_cast<int>(threadIdx.x));
    return false;
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

// The issuing thread: S_i = q_i K^T and O_i += P_i V, block by block, the two M tiles
// in turn.  nb0, nb1: blocks of each tile.
template <typename T>
__device__ __forceinline__ void issue_products(Control *ctl, uint8_t *q_smem, uint8_t *ring, uint32_t tmem, int nb0,
                                               int nb1, DeviceError *err) {
    using S = Shape<T>;
    const int nb = max(nb0, nb1);
    constexpr uint32_t qk_desc = f16_idesc(kTile, kKeys, false);
    constexpr uint32_t pv_desc = f16_idesc(kTile, kHeadDim, true);
    const uint32_t q_addr = smem_u32(q_smem);
    const uint32_t ring_addr = smem_u32(ring);
    auto full = [&](int seq) {
        return wait_for(&ctl->kv_full[seq % S::kRing], (seq / S::kRing) & 1, err);
    };
    auto logits = [&](int i, int seq) {  // S_i = q_i K^T
        const uint32_t kb = ring_addr + (seq % S::kRing) * kTileBytes;
#pragma unroll
        for (int part = 0; part < S::kParts; ++part) {
            const uint32_t qa = q_addr + (i * S::kParts + part) * kTileBytes;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t step = (k >> 2) * (kTileBytes / 2) + (k & 3) * 32;
                mma_ss(tmem + i * kKeys, smem_desc(qa + step, 16, 1024), smem_desc(kb + step, 16, 1024), qk_desc,
                       part > 0 || k > 0);
            }
        }
        tc_commit(smem_u32(&ctl->s_full[i]));
    };
    auto weigh = [&](int i, int seq, bool accumulate) {  // O_i += P_i V
        const uint32_t vb = ring_addr + (seq % S::kRing) * kTileBytes;
#pragma unroll
        for (int part = 0; part < S::kParts; ++part) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t p = tmem + i * kKeys + (k >> 1) * 32 + part * 16 + (k & 1) * 8;
                mma_ts(tmem + 256 + i * kHeadDim, p, smem_desc(vb + k * 2048, kTileBytes / 2, 1024), pv_desc,
                       accumulate || part > 0 || k > 0);
            }
        }
    };
    const int n_blocks[2] = {nb0, nb1};
    bool ok = nb > 0 && wait_for(&ctl->q_full, 0, err) && full(0);
    if (ok) {
        for (int i = 0; i < 2; ++i) {
            if (n_blocks[i] > 0) {
                logits(i, 0);
            }
        }
        tc_commit(smem_u32(&ctl->kv_empty[0]));
    }
    for (int j = 0; ok && j < nb; ++j) {
        const int v_seq = 2 * j + 1;
        ok = full(v_seq) && (j + 1 >= nb || full(v_seq + 1));
        for (int i = 0; ok && i < 2; ++i) {
            if (j >= n_blocks[i]) {
                continue;
            }
            ok = wait_for(&ctl->p_full[i], j & 1, err);
            if (!ok) {
                break;
            }
            tc_fence_after();
            weigh(i, v_seq, j > 0);
            if (j + 1 < n_blocks[i]) {
                logits(i, v_seq + 1);
            } else {
                tc_commit(smem_u32(&ctl->o_full[i]));
            }
        }
        if (ok) {
            tc_commit(smem_u32(&ctl->kv_empty[v_seq % S::kRing]));
            if (j + 1 < nb) {
                tc_commit(smem_u32(&ctl->kv_empty[(v_seq + 1) % S::kRing]));
            }
        }
    }
    if (!ok && nb > 0) {
        // products in flight end before the memory they use is given up
        tc_commit(smem_u32(&ctl->drained));
        mbar_wait_bounded(smem_u32(&ctl->drained), 0);
    }
}

template <typename T, bool kE4m3>
__global__ void __launch_bounds__(kThreads, 1)
    window_kernel(PoolView pool, const WindowTile *__restrict__ tiles, const int32_t *__restrict__ pages, int layer,
                  const T *__restrict__ q, int64_t q_stride, T *__restrict__ out, int64_t out_stride,
                  float *__restrict__ work, float scale_log2, DeviceError *err) {
    using S = Shape<T>;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t *q_smem = smem;
    uint8_t *ring = smem + S::kQBytes;
    Control *ctl = reinterpret_cast<Control *>(smem + S::kQBytes + S::kRing * kTileBytes);
    const WindowTile t = tiles[blockIdx.x];
    const int h = blockIdx.y;
    const int G = pool.n_head_kv;
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int n_tiles = t.tokens > kTileTokens ? 2 : 1;
    // 128-key blocks of each M tile: up to the last key that its last token sees
    const int key_end0 = t.pos0 + min(t.tokens, kTileTokens) - t.key0;
    const int nb0 = min(t.blocks, max(0, (key_end0 + kKeys - 1) / kKeys));
    const int nb1 = n_tiles == 2 ? t.blocks : 0;
    const int nb = max(nb0, nb1);

    if (warp == kIssuer) {
        tmem_alloc(smem_u32(&ctl->tmem), 512);
    }
    if (threadIdx.x == 0) {
        mbar_init(smem_u32(&ctl->q_full), kSoftmaxThreads);
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&ctl->s_full[i]), 1);
            mbar_init(smem_u32(&ctl->p_full[i]), kTile);
            mbar_init(smem_u32(&ctl->o_full[i]), 1);
        }
        for (int i = 0; i < S::kRing; ++i) {
            mbar_init(smem_u32(&ctl->kv_full[i]), kLoaderThreads);
            mbar_init(smem_u32(&ctl->kv_empty[i]), 1);
        }
        mbar_init(smem_u32(&ctl->drained), 1);
        ctl->odd_v = 0;
        fence_barrier_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctl->tmem;

    if (warp < 8) {
        // ------------------------------------------------------------ softmax
        const int i = warp >> 2;                      // M tile
        const int row = (warp & 3) * 32 + lane;       // = 4 token + head
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t s_col = tmem + lanes + i * kKeys;
        const uint32_t o_col = tmem + lanes + 256 + i * kHeadDim;
        // q: rows past the last token are zeros
        for (int it = 0; it < 16; ++it) {
            const int idx = it * kTile + row;
            const int r = idx >> 4;
            const int c = idx & 15;
            const int tok = i * kTileTokens + (r >> 2);
            float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (tok < t.tokens) {
                load8(q + (static_cast<int64_t>(t.row0) + tok) * q_stride + (kGqa * h + (r & 3)) * kHeadDim + c * 8, x);
            }
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                hi[k] = half2_bits(x[2 * k], x[2 * k + 1]);
                const float2 f = half2_floats(hi[k]);
                lo[k] = half2_bits(__fsub_rn(x[2 * k], f.x), __fsub_rn(x[2 * k + 1], f.y));
            }
            const uint32_t at = smem_u32(q_smem) + i * S::kParts * kTileBytes + tile_offset(kTile, r, c);
            st_shared16(at, hi[0], hi[1], hi[2], hi[3]);
            if (S::kSplit) {
                st_shared16(at + kTileBytes, lo[0], lo[1], lo[2], lo[3]);
            }
        }
        fence_proxy_async_smem();
        mbar_arrive(smem_u32(&ctl->q_full));

        const int my_tok = i * kTileTokens + (row >> 2);
        const int my_last = t.pos0 + min(my_tok, t.tokens - 1) - t.key0;  // last key this row sees
        const int first_last = t.pos0 + i * kTileTokens - t.key0;         // and the tile's first row
        const int blocks = i == 0 ? nb0 : nb1;
        float m = -INFINITY, l = 0.f;
        int e_v = kE4m3 ? kExpMin : 0;
        bool ok = true;
        for (int j = 0; j < blocks; ++j) {
            if (!__all_sync(0xffffffffu, wait_for(&ctl->s_full[i], j & 1, err))) {
                ok = false;
                break;
            }
            tc_fence_after();
            float s[kKeys];
            tmem_load128(s_col, s);
            const float *ks = ctl->k_scale[j % kScaleSlots];
            const int *ve = ctl->v_exp[j % kScaleSlots];
            if (j * kKeys + kKeys - 1 > first_last) {
                const int lim = my_last - j * kKeys;  // columns 0 .. lim are seen
#pragma unroll
                for (int k = 0; k < kKeys; ++k) {
                    s[k] = k <= lim ? s[k] : -INFINITY;
                }
            }
            float mx = -INFINITY;
#pragma unroll
            for (int p = 0; p < kBlockPages; ++p) {
                float a = s[16 * p], b = s[16 * p + 1];
#pragma unroll
                for (int k = 2; k < 16; k += 2) {
                    a = fmaxf(a, s[16 * p + k]);
                    b = fmaxf(b, s[16 * p + k + 1]);
                }
                mx = fmaxf(mx, fmaxf(a, b) * ks[p]);
            }
            // the bound and E move (o has to follow) only when they must
            int e_new = e_v;
            bool far = false;
            if (kE4m3) {
#pragma unroll
                for (int p = 0; p < kBlockPages; ++p) {
                    e_new = max(e_new, ve[p]);
                }
#pragma unroll
                for (int p = 0; p < kBlockPages; ++p) {
                    far = far || (ve[p] != kNoPage && ve[p] < e_new - kFar);
                }
            }
            const bool move = mx > m + kSlack || e_new > e_v;
            if (__any_sync(0xffffffffu, move)) {
                const float m_new = fmaxf(m, mx);
                const float corr = (m_new == -INFINITY ? 1.f : exp2_fast(m - m_new));
                const float o_corr = corr * pow2(max(e_v - e_new, -126));
                m = m_new;
                e_v = e_new;
                l *= corr;
                if (j > 0) {
#pragma unroll 1
                    for (int c = 0; c < kHeadDim; c += 16) {
                        float o[16];
                        tmem_load16(o_col + c, o);
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            o[k] *= o_corr;
                        }
                        tmem_store16(o_col + c, reinterpret_cast<const uint32_t (&)[16]>(o));
                    }
                }
            }
            const float bound = (m == -INFINITY ? 0.f : m) - kShift;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    // 2^(eV - E) belongs to the weight and not to l: in the exponent, and
                    // taken out of the page's sum again; where that could underflow
                    // (V pages 2^60 apart), by a product instead
                    const int page = 2 * c + p;
                    const float scale = ks[page];
                    const int d = kE4m3 && ve[page] != kNoPage ? ve[page] - e_v : 0;
                    const float off = (kE4m3 && !far ? static_cast<float>(d) : 0.f) - bound;
                    float *x = s + 16 * page;
                    float sum = 0.f, sum2 = 0.f;
#pragma unroll
                    for (int k = 0; k < 16; k += 2) {
                        x[k] = exp2_fast(fmaf(x[k], scale, off));
                        x[k + 1] = exp2_fast(fmaf(x[k + 1], scale, off));
                        sum += x[k];
                        sum2 += x[k + 1];
                    }
                    sum += sum2;
                    if (kE4m3) {
                        if (far) {
                            const float w = pow2(max(d, -126));
#pragma unroll
                            for (int k = 0; k < 16; ++k) {
                                x[k] *= w;
                            }
                            l += sum;
                        } else {
                            l = fmaf(sum, pow2(-d), l);
                        }
                    } else {
                        l += sum;
                    }
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        hi[8 * p + k] = half2_bits(x[2 * k], x[2 * k + 1]);
                        if (S::kSplit) {
                            const float2 f = half2_floats(hi[8 * p + k]);
                            lo[8 * p + k] = half2_bits(x[2 * k] - f.x, x[2 * k + 1] - f.y);
                        }
                    }
                }
                // in place of the logits: 16 columns of hi, 16 of lo per 32 keys
                tmem_store16(s_col + 32 * c, hi);
                if (S::kSplit) {
                    tmem_store16(s_col + 32 * c + 16, lo);
                }
            }
            tmem_store_wait();
            tc_fence_before();
            mbar_arrive(smem_u32(&ctl->p_full[i]));
        }
        if (ok && blocks > 0) {
            ok = __all_sync(0xffffffffu, wait_for(&ctl->o_full[i], 0, err));
        }
        if (ok) {
            tc_fence_after();
            const bool live = my_tok < t.tokens;
            const bool odd = *reinterpret_cast<volatile int *>(&ctl->odd_v) != 0;
            // a part's o is not normalised; o carries 2^kShift as l does
            const float f = pow2(max(e_v, -126)) * (t.part < 0 ? 1.f / l : 1.f);
            T *dst = out + (static_cast<int64_t>(t.row0) + my_tok) * out_stride + (kGqa * h + (row & 3)) * kHeadDim;
            float *part = work + (static_cast<int64_t>(t.part) * G + h) * kWindowPartFloats;
            for (int c = 0; c < 4; ++c) {
                float o[32];
                if (blocks > 0) {
                    tmem_load32(o_col + 32 * c, o);
                } else {
#pragma unroll
                    for (int k = 0; k < 32; ++k) {
                        o[k] = 0.f;
                    }
                }
#pragma unroll
                for (int k = 0; k < 32; ++k) {
                    o[k] = blocks > 0 ? o[k] * f : 0.f;
                }
                if (odd && live) {
                    const int keys = min(my_last + 1, t.blocks * kKeys);
                    for (int key = 0; key < keys; ++key) {
                        const int64_t page = pages[t.page_off + (t.key0 + key) / kPageTokens];
                        if (page < 0 || page >= pool.n_pages) {
                            continue;
                        }
#pragma unroll 1
                        for (int k = 0; k < 32; ++k) {
                            const float x = cached_value<kE4m3>(pool, page, layer, 1, h, key & 15, 32 * c + k);
                            if (!(fabsf(x) <= 3.402823466e38f)) {
#pragma unroll
                                for (int z = 0; z < 32; ++z) {
                                    o[z] += z == k ? x : 0.f;
                                }
                            }
                        }
                    }
                }
                if (t.part >= 0) {
                    for (int k = 0; k < 32; k += 4) {
                        store4(part + (i * kTile + row) * kHeadDim + 32 * c + k, o + k);
                    }
                } else if (live) {
                    for (int k = 0; k < 32; k += 4) {
                        store4(dst + 32 * c + k, o + k);
                    }
                }
            }
            if (t.part >= 0) {
                float2 *ml = reinterpret_cast<float2 *>(part + kWindowTokens * kGqa * kHeadDim);
                ml[i * kTile + row] = make_float2(m, l);
            }
            tc_fence_before();
        }
    } else if (warp < kIssuer) {
        // ------------------------------------------------------------ loaders
        const int tid = threadIdx.x - kSoftmaxThreads;
        const int n_pages = (t.pos0 + t.tokens - 1) / kPageTokens + 1;  // of the slot, up to its last key here
        // A block is filled in steps of 1024 16-byte pieces: K, V (8-bit cache) or the
        // two halves of K, then of V (F16).  Two steps' pieces are in registers: a
        // step's loads go out when the step two before it is stored.  A piece: 8 bits,
        // 16 dims of a row of one of 8 pages; F16, 8 dims of a row of one of 4.
        // Eight consecutive threads store to eight different bank groups: 8 bits, dims
        // 0-63 or 64-127 of two neighbouring rows (an even and an odd row's swizzles
        // interleave); F16, half a row.
        constexpr int kSteps = kE4m3 ? 2 : 4;
        constexpr int kAhead = 2;
        constexpr int kPieces = 1024;
        constexpr int kEach = (kPieces + kLoaderThreads - 1) / kLoaderThreads;
        static_assert(kLoaderThreads % 16 == 0, "a thread keeps its place in the row");
        const int c = kE4m3 ? ((tid >> 3) & 1) * 4 + (tid & 3) : tid & 15;  // piece of the row
        const int row0 = kE4m3 ? 2 * (tid >> 4) + ((tid >> 2) & 1) : tid >> 4;
        constexpr int kRowStep = (kE4m3 ? 2 : 1) * kLoaderThreads / 16;
        const int64_t page_stride = static_cast<int64_t>(G) * cache_unit_bytes(pool.format);
        const uint8_t *base = pool.base + static_cast<int64_t>(layer) * pool.n_pages * page_stride +
                              h * (kE4m3 ? kCodeUnitBytes : kHeadBlockBytes);
        const int64_t v_off = kE4m3 ? kCodeBlockBytes : static_cast<int64_t>(G) * kHeadBlockBytes;
        const int32_t *list = pages + t.page_off + t.key0 / kPageTokens;
        const int last_page = n_pages - 1 - t.key0 / kPageTokens;
        int bad = -1;
        // Past the slot's pages its last one is read again: K there is masked, V zeroed.
        auto page_at = [&](int index) {
            int page = list[min(index, last_page)];
            if (page >= pool.n_pages || page < 0) {
                bad = index;
                page = 0;
            }
            return page;
        };
        uint4 raw[kAhead][kEach];
        auto fetch = [&](int j, int step, uint4 (&to)[kEach]) {
            const uint8_t *from = base + (step * 2 / kSteps == 1 ? v_off : 0);
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
        const int last_key = t.pos0 + t.tokens - 1 - t.key0;
        auto put = [&](int j, int step, const uint4 (&from)[kEach], uint32_t buf) {
            const bool is_v = step * 2 / kSteps == 1;
            const bool tail = is_v && j * kKeys + kKeys - 1 > last_key;
            bool odd = false;
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const int row = (kE4m3 ? 0 : 64 * (step & 1)) + row0 + i * kRowStep;
                if (i == kEach - 1 && tid + i * kLoaderThreads >= kPieces) {
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
                *reinterpret_cast<volatile int *>(&ctl->odd_v) = 1;
            }
        };
        // The exponents of a block's K and V, with its K tile: thread p takes page p's.
        int2 exps = make_int2(0, kNoPage);
        auto fetch_exponents = [&](int j) {
            if (kE4m3 && tid < kBlockPages) {
                const int index = j * kBlockPages + tid;
                exps = *reinterpret_cast<const int2 *>(base + page_at(index) * page_stride + 2 * kCodeBlockBytes);
                if (index > last_page) {
                    exps.y = kNoPage;
                }
            }
        };
        fetch(0, 0, raw[0]);
        fetch(0, 1, raw[1]);
        fetch_exponents(0);
        bool ok = true;
        for (int j = 0; ok && j < nb; ++j) {
#pragma unroll
            for (int step = 0; step < kSteps; ++step) {
                const int seq = 2 * j + step * 2 / kSteps;  // the operand tile
                const int slot = seq % S::kRing;
                const bool first_step = step % (kSteps / 2) == 0;
                const bool last_step = (step + 1) % (kSteps / 2) == 0;
                if (first_step && seq >= S::kRing) {
                    ok = ok && wait_for(&ctl->kv_empty[slot], (seq / S::kRing - 1) & 1, err);
                }
                if (!ok) {
                    break;
                }
                if (step == 0 && tid < kBlockPages) {
                    ctl->k_scale[j % kScaleSlots][tid] = scale_log2 * pow2(exps.x);
                    ctl->v_exp[j % kScaleSlots][tid] = exps.y;
                }
                put(j, step, raw[step % kAhead], smem_u32(ring) + slot * kTileBytes);
                if (last_step) {
                    fence_proxy_async_smem();
                    mbar_arrive(smem_u32(&ctl->kv_full[slot]));
                }
                if (step + kAhead < kSteps) {
                    fetch(j, step + kAhead, raw[step % kAhead]);
                } else if (j + 1 < nb) {
                    fetch(j + 1, step + kAhead - kSteps, raw[step % kAhead]);
                    if (step + kAhead == kSteps) {
                        fetch_exponents(j + 1);
                    }
                }
            }
        }
        if (bad >= 0) {
            record(err, kErrBadIndex, list[min(bad, last_page)], bad);
        }
    } else {
        // ----------------------------------------------------------- products
        if (lane == 0) {
            issue_products<T>(ctl, q_smem, ring, tmem, nb0, nb1, err);
        }
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
        cudaFuncSetAttribute(window_kernel<T, kE4m3>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<T>::kSmem);
        if (dev >= 0 && dev < 64) {
            configured[dev] = true;
        }
    }
    const unsigned G = static_cast<unsigned>(pool.n_head_kv);
    T *out = static_cast<T *>(a.out);
    window_kernel<T, kE4m3><<<dim3(static_cast<unsigned>(a.n_tiles), G), kThreads, Shape<T>::kSmem, stream>>>(
        pool, a.tiles, a.pages, a.layer, static_cast<const T *>(a.q), a.q_stride, out, a.out_stride, a.work,
        a.scale_log2, err);
    if (a.n_merges > 0) {
        window_combine_kernel<T>
            <<<dim3(static_cast<unsigned>(a.n_merges), G, kWindowTokens * kGqa / 8), 256, 0, stream>>>(
                a.merges, static_cast<int>(G), a.work, out, a.out_stride);
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
