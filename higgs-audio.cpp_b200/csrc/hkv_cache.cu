// hkv_cache.cu -- rows into the paged cache and back, for both cache formats.
//
//   write_kernel  one CTA per (page item, KV head): the K row, the V row and the
//                 four query rows of every token of the item.  Per-head RMS norm
//                 (optional), NEOX rotation of q and k, then q to q_out, K and V
//                 into the page.  Sixteen lanes hold a row, lane l dims 4l .. 4l + 3 and
//                 64 + 4l .. 64 + 4l + 3: both partners of a rotation, which then
//                 needs no exchange, and each cosine once.  They are read once for a
//                 token's five rotated rows.  In the 8-bit format the CTA owns the
//                 whole blocks of K and V, so their exponents need one exchange
//                 through shared memory, and the rows that were there are rounded
//                 again by the lanes whose row it is.
//   read_kernel   rows of the cache as F16 or F32 values, packed.
//
// Both are bound by their bytes for prompts (an F32 row of K and V is 8 KiB in,
// 2 KiB out) and by the launch and one chain of loads for single tokens.  Measured on the
// 8-bit cache: 12 ragged prompts, 11,668 packed BF16 rows with norms, written in 53.7 us (0.76
// of the copy rate: 8-byte loads of 16-bit rows, 4-byte stores of codes) and read back as
// F16 in 14.7 (0.76); 1500 F32 rows 5.8 and 3.0 us; 32 slots of one F32 token 2.3 and
// 1.6.  On the F16 cache 48.0 (0.93) and 17.9, 3.9 and 3.0, 2.2 and 1.6.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "hkv_device.cuh"
#include "hkv_e4m3.cuh"
#include "hkv_internal.h"

namespace hkv {
namespace {

using namespace dev;

constexpr int kWhereWrite = 6;
constexpr int kWhereRead = 7;
constexpr int kDtypeF32 = 0;
constexpr int kDtypeF16 = 1;

__device__ __forceinline__ void record(DeviceError *err, int where, int a, int b) {
    if (atomicCAS(&err->code, 0, kErrBadIndex) == 0) {
        err->where = where;
        err->a = a;
        err->b = b;
    }
}

// A lane's two runs of four elements, 64 apart, raw and as F32.  Plain loads: q_out
// may be q itself, each row of a head being read and written by the same lanes.
struct Raw32 {
    float4 a, b;
};
struct Raw16 {
    uint2 a, b;
};
__device__ __forceinline__ Raw32 load_row(const float *p) {
    return {*reinterpret_cast<const float4 *>(p), *reinterpret_cast<const float4 *>(p + 64)};
}
__device__ __forceinline__ Raw16 load_row(const __half *p) {
    return {*reinterpret_cast<const uint2 *>(p), *reinterpret_cast<const uint2 *>(p + 64)};
}
__device__ __forceinline__ Raw16 load_row(const __nv_bfloat16 *p) {
    return {*reinterpret_cast<const uint2 *>(p), *reinterpret_cast<const uint2 *>(p + 64)};
}
__device__ __forceinline__ void unpack(const Raw32 &r, const float *, float (&x)[8]) {
    x[0] = r.a.x; x[1] = r.a.y; x[2] = r.a.z; x[3] = r.a.w;
    x[4] = r.b.x; x[5] = r.b.y; x[6] = r.b.z; x[7] = r.b.w;
}
__device__ __forceinline__ void unpack(const Raw16 &r, const __half *, float (&x)[8]) {
    const uint32_t w[4] = {r.a.x, r.a.y, r.b.x, r.b.y};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void unpack(const Raw16 &r, const __nv_bfloat16 *, float (&x)[8]) {
    const uint32_t w[4] = {r.a.x, r.a.y, r.b.x, r.b.y};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ uint32_t half_pair(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ void store_row(float *p, const float (&x)[8]) {
    *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4 *>(p + 64) = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store_row(__half *p, const float (&x)[8]) {
    *reinterpret_cast<uint2 *>(p) = make_uint2(half_pair(x[0], x[1]), half_pair(x[2], x[3]));
    *reinterpret_cast<uint2 *>(p + 64) = make_uint2(half_pair(x[4], x[5]), half_pair(x[6], x[7]));
}
__device__ __forceinline__ void store_row(__nv_bfloat16 *p, const float (&x)[8]) {
    *reinterpret_cast<uint2 *>(p) = make_uint2(bf16_pair(x[0], x[1]), bf16_pair(x[2], x[3]));
    *reinterpret_cast<uint2 *>(p + 64) = make_uint2(bf16_pair(x[4], x[5]), bf16_pair(x[6], x[7]));
}

// RMS norm of a row held by 16 lanes.
__device__ __forceinline__ void norm_row(float (&x)[8], const float *weight, float eps, int lane) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        ss += x[i] * x[i];
    }
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) {
        ss += __shfl_xor_sync(0xffffffffu, ss, off);
    }
    const float inv = rsqrtf(ss * (1.f / kHeadDim) + eps);
    float g[8];
    unpack(load_row(weight + 4 * lane), weight, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[i] = x[i] * inv * g[i];
    }
}

// NEOX rotation.  Products and sums rounded one by one, as the append kernel
// of the F16 cache rounds them, so both formats quantise the same F32 rows.
__device__ __forceinline__ void rotate_row(float (&x)[8], const float4 &c4, const float4 &s4) {
    const float c[4] = {c4.x, c4.y, c4.z, c4.w};
    const float s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = x[i], b = x[4 + i];
        x[i] = __fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(b, s[i]));
        x[4 + i] = __fadd_rn(__fmul_rn(a, s[i]), __fmul_rn(b, c[i]));
    }
}

__device__ __forceinline__ float row_amax(const float (&x)[8]) {
    float a = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        a = fmaxf(a, finite_abs(x[i]));
    }
    return a;
}

// Byte of dims 4 lane .. 4 lane + 3 of row r in a code block, and of the run 64
// dims on.
__device__ __forceinline__ int code_offset(int r, int lane) {
    return r * kHeadDim + (((lane >> 2) ^ (r & 7)) << 4) + ((lane & 3) << 2);
}
constexpr int kCodeOffsetUpper = 64;  // chunk c + 4 lies at (c + 4) ^ (r & 7) = (c ^ (r & 7)) ^ 4
__device__ __forceinline__ void put_codes(uint8_t *block, int r, int lane, const float (&x)[8], float inv) {
    const int at = code_offset(r, lane);
    *reinterpret_cast<uint32_t *>(block + at) = to_codes4(make_float4(x[0], x[1], x[2], x[3]), inv);
    *reinterpret_cast<uint32_t *>(block + (at ^ kCodeOffsetUpper)) =
        to_codes4(make_float4(x[4], x[5], x[6], x[7]), inv);
}
__device__ __forceinline__ void rescale_row(uint8_t *block, int r, int lane, int d) {
    const int at = code_offset(r, lane);
    uint32_t *lo = reinterpret_cast<uint32_t *>(block + at);
    uint32_t *hi = reinterpret_cast<uint32_t *>(block + (at ^ kCodeOffsetUpper));
    *lo = rescale_codes4(*lo, d);
    *hi = rescale_codes4(*hi, d);
}
__device__ __forceinline__ void put_f16(uint8_t *block, int r, int lane, const float (&x)[8]) {
    uint8_t *row = block + r * kRowBytes + (lane & 1) * 8;
    *reinterpret_cast<uint2 *>(row + swizzled_chunk(r, lane >> 1) * 16) =
        make_uint2(half_pair(x[0], x[1]), half_pair(x[2], x[3]));
    *reinterpret_cast<uint2 *>(row + swizzled_chunk(r, 8 + (lane >> 1)) * 16) =
        make_uint2(half_pair(x[4], x[5]), half_pair(x[6], x[7]));
}

// kOneRow: items of one row (the tokens of a decode batch); the six rows of a
// (token, KV head) then go to six half-warps, so that no lane idles for fifteen
// absent rows.  Otherwise half-warp r holds row r of the page and takes K, V and
// the query rows in turn.
template <typename T, bool kE4m3, bool kOneRow>
__global__ void __launch_bounds__(kOneRow ? 96 : 256, kOneRow ? 1 : sizeof(T) == 4 ? 4 : 5)
    write_kernel(PoolView pool, RopeView rope, BatchView batch, WriteArgs a, DeviceError *err) {
    using Raw = decltype(load_row(static_cast<const T *>(nullptr)));
    __shared__ float s_amax[2][16];
    pdl_wait();
    pdl_trigger();
    const int G = pool.n_head_kv;
    const int item = blockIdx.x / G;
    const int head = blockIdx.x - item * G;
    RowItem it;
    if (a.items != nullptr) {
        it = a.items[item];
    } else {
        it.pos0 = batch.pos[item];
        it.page = batch.pages[batch.page_off[item] + (it.pos0 >> 4)];
        it.row0 = item;
        it.count = 1;
    }
    const int r0 = it.pos0 & 15;
    if (it.page < 0 || it.page >= pool.n_pages || it.pos0 < 0 || it.count < 1 ||
        r0 + it.count > kPageTokens || it.pos0 + it.count > rope.context_length || (kOneRow && it.count != 1)) {
        if (threadIdx.x == 0) {
            record(err, kWhereWrite, it.page, it.pos0);
        }
        return;
    }
    const int lane = threadIdx.x & 15;
    const int hw = threadIdx.x >> 4;
    const int r = kOneRow ? r0 : hw;  // row of the page
    const bool live = r >= r0 && r < r0 + it.count;
    const int64_t row = it.row0 + (live ? r - r0 : 0);
    const bool has_q = a.q != nullptr;
    const T *kp = static_cast<const T *>(a.k) + row * a.k_stride + head * kHeadDim + 4 * lane;
    const T *vp = static_cast<const T *>(a.v) + row * a.v_stride + head * kHeadDim + 4 * lane;
    const T *qp = has_q ? static_cast<const T *>(a.q) + row * a.q_stride + kGqa * head * kHeadDim + 4 * lane : kp;
    T *qo = has_q ? static_cast<T *>(a.q_out) + row * a.q_out_stride + kGqa * head * kHeadDim + 4 * lane : nullptr;
    uint8_t *k_block, *v_block;
    int *exps = nullptr;
    int e_old[2] = {kExpMin, kExpMin};
    if (kE4m3) {
        k_block = pool.base + code_unit_index(it.page, a.layer, head, pool.n_pages, G) * kCodeUnitBytes;
        v_block = k_block + kCodeBlockBytes;
        exps = reinterpret_cast<int *>(k_block + 2 * kCodeBlockBytes);
        if (r0 > 0) {  // the rows before r0 are held under these
            e_old[0] = exps[0];
            e_old[1] = exps[1];
        }
    } else {
        k_block = pool.base + head_block_index(it.page, a.layer, 0, head, pool.n_pages, G) * kHeadBlockBytes;
        v_block = k_block + static_cast<int64_t>(G) * kHeadBlockBytes;
    }
    float4 cs = make_float4(1.f, 1.f, 1.f, 1.f), sn = make_float4(0.f, 0.f, 0.f, 0.f);
    if (a.rope) {
        const int64_t at = static_cast<int64_t>(it.pos0 - r0 + (live ? r : r0)) * (kHeadDim / 2) + 4 * lane;
        cs = *reinterpret_cast<const float4 *>(rope.cos_tab + at);
        sn = *reinterpret_cast<const float4 *>(rope.sin_tab + at);
    }
    auto finish = [&](float (&x)[8], const float *norm) {
        if (norm != nullptr) {
            norm_row(x, norm, a.eps, lane);
        }
        if (a.rope) {
            rotate_row(x, cs, sn);
        }
    };
    if (kOneRow) {
        const int slice = hw;
        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (slice < 2 || has_q) {
            const T *src = slice == 0 ? kp : slice == 1 ? vp : qp + (slice - 2) * kHeadDim;
            unpack(load_row(src), src, x);
        }
        // the half-warps of a warp take the norm's shuffles together; V keeps its own
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            y[i] = x[i];
        }
        finish(y, slice < 2 ? a.k_norm : a.q_norm);
        if (slice != 1) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = y[i];
            }
        }
        if (slice >= 2) {
            if (has_q) {
                store_row(qo + (slice - 2) * kHeadDim, x);
            }
            return;
        }
        uint8_t *block = slice == 0 ? k_block : v_block;
        if (!kE4m3) {
            put_f16(block, r0, lane, x);
            return;
        }
        float amax = row_amax(x);
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) {
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
        }
        const int old = slice == 0 ? e_old[0] : e_old[1];
        const int e = max(block_exponent(amax), old);
        if (r0 > 0 && e > old) {
            for (int other = 0; other < kPageTokens; ++other) {
                if (other != r0) {
                    rescale_row(block, other, lane, e - old);
                }
            }
        }
        put_codes(block, r0, lane, x, pow2(-e));
        __syncwarp();  // every lane has its old exponent
        if (lane == 0) {
            exps[slice] = e;
        }
        return;
    }
    // K, V and the first two query rows are loaded at once, the other two while
    // those are worked on: more in flight would cost a resident CTA its registers
    Raw rk = {}, rv = {}, rq[2] = {};
    if (live) {
        rk = load_row(kp);
        rv = load_row(vp);
        if (has_q) {
            rq[0] = load_row(qp);
            rq[1] = load_row(qp + kHeadDim);
        }
    }
    float k[8], v[8];
    unpack(rk, kp, k);
    unpack(rv, vp, v);
    finish(k, a.k_norm);
    if (kE4m3) {
        float ak = row_amax(k), av = row_amax(v);
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) {
            ak = fmaxf(ak, __shfl_xor_sync(0xffffffffu, ak, off));
            av = fmaxf(av, __shfl_xor_sync(0xffffffffu, av, off));
        }
        if (lane == 0) {
            s_amax[0][hw] = live ? ak : 0.f;
            s_amax[1][hw] = live ? av : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            float amax = s_amax[side][lane];
#pragma unroll
            for (int off = 8; off > 0; off >>= 1) {
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
            }
            const int e = max(block_exponent(amax), e_old[side]);
            uint8_t *block = side ? v_block : k_block;
            if (live) {
                put_codes(block, r, lane, side ? v : k, pow2(-e));
            } else if (r0 > 0 && e > e_old[side]) {
                rescale_row(block, r, lane, e - e_old[side]);
            }
            if (threadIdx.x == 0) {
                exps[side] = e;
            }
        }
    } else if (live) {
        put_f16(k_block, r, lane, k);
        put_f16(v_block, r, lane, v);
    }
    if (has_q) {
#pragma unroll
        for (int pair = 0; pair < 2; ++pair) {
            float x[8], y[8];
            unpack(rq[0], qp, x);
            unpack(rq[1], qp, y);
            if (pair == 0 && live) {
                rq[0] = load_row(qp + 2 * kHeadDim);
                rq[1] = load_row(qp + 3 * kHeadDim);
            }
            finish(x, a.q_norm);
            finish(y, a.q_norm);
            if (live) {
                store_row(qo + 2 * pair * kHeadDim, x);
                store_row(qo + (2 * pair + 1) * kHeadDim, y);
            }
        }
    }
}

// A launch that may be set up while the kernel before it runs: the kernel waits
// (griddepcontrol.wait) before its first load.
template <typename Kernel, typename... Args>
void launch_dependent(Kernel kernel, unsigned blocks, unsigned threads, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <typename T, bool kE4m3>
void launch_write_t(const PoolView &pool, const RopeView &rope, const BatchView &batch,
                    const WriteArgs &a, DeviceError *err, cudaStream_t stream) {
    const unsigned blocks = static_cast<unsigned>(a.n_items) * static_cast<unsigned>(pool.n_head_kv);
    if (a.one_row) {
        launch_dependent(write_kernel<T, kE4m3, true>, blocks, 96, stream, pool, rope, batch, a, err);
    } else {
        launch_dependent(write_kernel<T, kE4m3, false>, blocks, 256, stream, pool, rope, batch, a, err);
    }
}

// ======================================================================== read
// One CTA per (page item, KV head, K or V), 16 lanes a row.
template <typename T, bool kE4m3>
__global__ void __launch_bounds__(256)
    read_kernel(PoolView pool, const RowItem *__restrict__ items, int layer, T *__restrict__ k_out,
                T *__restrict__ v_out, DeviceError *err) {
    pdl_wait();
    pdl_trigger();
    const int G = pool.n_head_kv;
    const int item = blockIdx.x / (2 * G);
    const int side = blockIdx.x - item * 2 * G;
    const int kv = side >= G ? 1 : 0;
    const int head = side - kv * G;
    const RowItem it = items[item];
    const int r0 = it.pos0 & 15;
    if (it.page < 0 || it.page >= pool.n_pages || it.count < 1 || r0 + it.count > kPageTokens) {
        if (threadIdx.x == 0) {
            record(err, kWhereRead, it.page, it.pos0);
        }
        return;
    }
    const int lane = threadIdx.x & 15;
    const int r = threadIdx.x >> 4;
    if (r >= it.count) {
        return;
    }
    const int row = r0 + r;
    float x[8];
    if (kE4m3) {
        const uint8_t *unit = pool.base + code_unit_index(it.page, layer, head, pool.n_pages, G) * kCodeUnitBytes;
        const int e = reinterpret_cast<const int *>(unit + 2 * kCodeBlockBytes)[kv];
        const int at = kv * kCodeBlockBytes + code_offset(row, lane);
        const float4 lo = codes_to_float4(*reinterpret_cast<const uint32_t *>(unit + at));
        const float4 hi = codes_to_float4(*reinterpret_cast<const uint32_t *>(unit + (at ^ kCodeOffsetUpper)));
        const float scale = pow2(e);
        x[0] = lo.x * scale; x[1] = lo.y * scale; x[2] = lo.z * scale; x[3] = lo.w * scale;
        x[4] = hi.x * scale; x[5] = hi.y * scale; x[6] = hi.z * scale; x[7] = hi.w * scale;
    } else {
        const uint8_t *p =
            pool.base + head_block_index(it.page, layer, kv, head, pool.n_pages, G) * kHeadBlockBytes +
            row * kRowBytes + (lane & 1) * 8;
        const Raw16 raw = {*reinterpret_cast<const uint2 *>(p + swizzled_chunk(row, lane >> 1) * 16),
                           *reinterpret_cast<const uint2 *>(p + swizzled_chunk(row, 8 + (lane >> 1)) * 16)};
        unpack(raw, static_cast<const __half *>(nullptr), x);
    }
    store_row((kv != 0 ? v_out : k_out) + (static_cast<int64_t>(it.row0 + r) * G + head) * kHeadDim + 4 * lane, x);
}

template <typename T>
void launch_read_t(const PoolView &pool, const RowItem *items, int32_t n_items, int layer, void *k_out,
                   void *v_out, DeviceError *err, cudaStream_t stream) {
    T *k = static_cast<T *>(k_out);
    T *v = static_cast<T *>(v_out);
    const unsigned blocks = static_cast<unsigned>(n_items) * 2 * static_cast<unsigned>(pool.n_head_kv);
    if (pool.format == kCacheE4m3) {
        launch_dependent(read_kernel<T, true>, blocks, 256, stream, pool, items, layer, k, v, err);
    } else {
        launch_dependent(read_kernel<T, false>, blocks, 256, stream, pool, items, layer, k, v, err);
    }
}

template <typename T>
void launch_write_f(const PoolView &pool, const RopeView &rope, const BatchView &batch, const WriteArgs &a,
                    DeviceError *err, cudaStream_t stream) {
    if (pool.format == kCacheE4m3) {
        launch_write_t<T, true>(pool, rope, batch, a, err, stream);
    } else {
        launch_write_t<T, false>(pool, rope, batch, a, err, stream);
    }
}

}  // namespace

void launch_write(const PoolView &pool, const RopeView &rope, const BatchView &batch,
                  const WriteArgs &args, DeviceError *err, cudaStream_t stream) {
    if (args.dtype == kDtypeF32) {
        launch_write_f<float>(pool, rope, batch, args, err, stream);
    } else if (args.dtype == kDtypeF16) {
        launch_write_f<__half>(pool, rope, batch, args, err, stream);
    } else {
        launch_write_f<__nv_bfloat16>(pool, rope, batch, args, err, stream);
    }
}

void launch_read(const PoolView &pool, const RowItem *items, int32_t n_items, int layer, int dtype,
                 void *k_out, void *v_out, DeviceError *err, cudaStream_t stream) {
    if (dtype == kDtypeF32) {
        launch_read_t<float>(pool, items, n_items, layer, k_out, v_out, err, stream);
    } else {
        launch_read_t<__half>(pool, items, n_items, layer, k_out, v_out, err, stream);
    }
}

}  // namespace hkv
