// hkv_cache.cu -- rows into the paged cache and back, for both cache formats.
//
//   write_kernel  one warp per (page item, head slice): up to 16 rows of one
//                 query, key or value head, 4 dims per lane.  Per-head RMS norm
//                 (optional), NEOX rotation of q and k, then q rows to q_out and
//                 K / V rows into the page.  In the 8-bit format the warp owns
//                 the whole (page, KV head, K or V) block, so the block's
//                 exponent, the rounding of the new rows and -- when a new row
//                 outgrows the exponent -- the second rounding of the rows that
//                 were there need no word from another warp.
//   read_kernel   rows of the cache as F16 or F32 values, packed.
//
// Both are bound by their bytes for prompts (an F32 row of K and V is 8 KiB in,
// 2 KiB out) and by the launch and one chain of loads for single tokens.
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

// Four consecutive elements.  Plain loads: q_out may be q itself, each row of a
// head being read and written by one warp.
__device__ __forceinline__ float4 load4(const float *p) {
    return *reinterpret_cast<const float4 *>(p);
}
__device__ __forceinline__ float4 load4(const __half *p) {
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&u.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&u.y));
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float4 load4(const __nv_bfloat16 *p) {
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u),
                       __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
}
__device__ __forceinline__ uint2 half4(float4 x) {
    const __half2 a = __floats2half2_rn(x.x, x.y), b = __floats2half2_rn(x.z, x.w);
    return make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}
__device__ __forceinline__ void store4(float *p, float4 x) { *reinterpret_cast<float4 *>(p) = x; }
__device__ __forceinline__ void store4(__half *p, float4 x) { *reinterpret_cast<uint2 *>(p) = half4(x); }
__device__ __forceinline__ void store4(__nv_bfloat16 *p, float4 x) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(x.x, x.y), b = __floats2bfloat162_rn(x.z, x.w);
    *reinterpret_cast<uint2 *>(p) =
        make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        x += __shfl_xor_sync(0xffffffffu, x, off);
    }
    return x;
}
__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off));
    }
    return x;
}

// Rotation of a row whose lane l holds dims 4l .. 4l + 3: the partner half is
// 16 lanes away.  Products and sums rounded one by one, as the append kernel
// of the F16 cache rounds them, so both formats quantise the same F32 rows.
__device__ __forceinline__ float4 rotate(float4 x, float4 c, float4 s, bool upper) {
    float4 p;
    p.x = __shfl_xor_sync(0xffffffffu, x.x, 16);
    p.y = __shfl_xor_sync(0xffffffffu, x.y, 16);
    p.z = __shfl_xor_sync(0xffffffffu, x.z, 16);
    p.w = __shfl_xor_sync(0xffffffffu, x.w, 16);
    float4 y;
    if (upper) {
        y.x = __fadd_rn(__fmul_rn(p.x, s.x), __fmul_rn(x.x, c.x));
        y.y = __fadd_rn(__fmul_rn(p.y, s.y), __fmul_rn(x.y, c.y));
        y.z = __fadd_rn(__fmul_rn(p.z, s.z), __fmul_rn(x.z, c.z));
        y.w = __fadd_rn(__fmul_rn(p.w, s.w), __fmul_rn(x.w, c.w));
    } else {
        y.x = __fsub_rn(__fmul_rn(x.x, c.x), __fmul_rn(p.x, s.x));
        y.y = __fsub_rn(__fmul_rn(x.y, c.y), __fmul_rn(p.y, s.y));
        y.z = __fsub_rn(__fmul_rn(x.z, c.z), __fmul_rn(p.z, s.z));
        y.w = __fsub_rn(__fmul_rn(x.w, c.w), __fmul_rn(p.w, s.w));
    }
    return y;
}

// Byte of dims 4 lane .. 4 lane + 3 of row r in a code block.
__device__ __forceinline__ int code_offset(int r, int lane) {
    return r * kHeadDim + (((lane >> 2) ^ (r & 7)) << 4) + ((lane & 3) << 2);
}

constexpr int kWriteWarps = 4;

template <typename T, bool kE4m3>
__global__ void __launch_bounds__(kWriteWarps * 32)
    write_kernel(PoolView pool, RopeView rope, BatchView batch, WriteArgs a, DeviceError *err) {
    const int lane = threadIdx.x & 31;
    const int G = pool.n_head_kv;
    const int slices = (2 + (a.q != nullptr ? kGqa : 0)) * G;
    const int64_t warp = static_cast<int64_t>(blockIdx.x) * kWriteWarps + (threadIdx.x >> 5);
    const int64_t item = warp / slices;
    const int slice = static_cast<int>(warp - item * slices);
    if (item >= a.n_items) {
        return;
    }
    RowItem it;
    if (a.items != nullptr) {
        it = a.items[item];
    } else {
        it.pos0 = batch.pos[item];
        it.page = batch.pages[batch.page_off[item] + (it.pos0 >> 4)];
        it.row0 = static_cast<int>(item);
        it.count = 1;
    }
    const int r0 = it.pos0 & 15;
    if (it.page < 0 || it.page >= pool.n_pages || it.pos0 < 0 || it.count < 1 ||
        r0 + it.count > kPageTokens || it.pos0 + it.count > rope.context_length) {
        if (lane == 0) {
            record(err, kWhereWrite, it.page, it.pos0);
        }
        return;
    }
    // slices: K heads, V heads, query heads
    const bool is_q = slice >= 2 * G;
    const bool is_v = !is_q && slice >= G;
    const int head = is_q ? slice - 2 * G : is_v ? slice - G : slice;
    const int64_t stride = is_q ? a.q_stride : is_v ? a.v_stride : a.k_stride;
    const T *src = static_cast<const T *>(is_q ? a.q : is_v ? a.v : a.k) + it.row0 * stride +
                   head * kHeadDim + 4 * lane;
    uint8_t *unit = nullptr;
    int *exp_slot = nullptr;
    int e_old = kExpMin;
    if (kE4m3 && !is_q) {
        unit = pool.base + code_unit_index(it.page, a.layer, head, pool.n_pages, G) * kCodeUnitBytes;
        exp_slot = reinterpret_cast<int *>(unit + 2 * kCodeBlockBytes) + (is_v ? 1 : 0);
        unit += is_v ? kCodeBlockBytes : 0;
        if (r0 > 0) {
            e_old = *exp_slot;  // the rows before r0 are held under it
        }
    }
    float4 x[kPageTokens];
#pragma unroll
    for (int r = 0; r < kPageTokens; ++r) {
        if (r < it.count) {
            x[r] = load4(src + r * stride);
        }
    }
    const float *norm = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
    if (norm != nullptr) {
        const float4 w = load4(norm + 4 * lane);
#pragma unroll
        for (int r = 0; r < kPageTokens; ++r) {
            if (r < it.count) {
                const float ss = warp_sum(x[r].x * x[r].x + x[r].y * x[r].y + x[r].z * x[r].z +
                                          x[r].w * x[r].w);
                const float inv = 1.f / sqrtf(ss * (1.f / kHeadDim) + a.eps);
                x[r].x = x[r].x * inv * w.x;
                x[r].y = x[r].y * inv * w.y;
                x[r].z = x[r].z * inv * w.z;
                x[r].w = x[r].w * inv * w.w;
            }
        }
    }
    if (a.rope && !is_v) {
        const float *cp = rope.cos_tab + static_cast<int64_t>(it.pos0) * (kHeadDim / 2) + ((4 * lane) & 63);
        const float *sp = rope.sin_tab + static_cast<int64_t>(it.pos0) * (kHeadDim / 2) + ((4 * lane) & 63);
#pragma unroll
        for (int r = 0; r < kPageTokens; ++r) {
            if (r < it.count) {
                x[r] = rotate(x[r], load4(cp + r * (kHeadDim / 2)), load4(sp + r * (kHeadDim / 2)),
                              lane >= 16);
            }
        }
    }
    if (is_q) {
        T *dst = static_cast<T *>(a.q_out) + it.row0 * a.q_out_stride + head * kHeadDim + 4 * lane;
#pragma unroll
        for (int r = 0; r < kPageTokens; ++r) {
            if (r < it.count) {
                store4(dst + r * a.q_out_stride, x[r]);
            }
        }
        return;
    }
    if (!kE4m3) {
        uint8_t *block = pool.base + head_block_index(it.page, a.layer, is_v ? 1 : 0, head, pool.n_pages, G) *
                                         kHeadBlockBytes;
#pragma unroll
        for (int r = 0; r < kPageTokens; ++r) {
            if (r < it.count) {
                const int row = r0 + r;
                *reinterpret_cast<uint2 *>(block + row * kRowBytes + swizzled_chunk(row, lane >> 1) * 16 +
                                           (lane & 1) * 8) = half4(x[r]);
            }
        }
        return;
    }
    float amax = 0.f;
#pragma unroll
    for (int r = 0; r < kPageTokens; ++r) {
        if (r < it.count) {
            amax = fmaxf(amax, fmaxf(fmaxf(finite_abs(x[r].x), finite_abs(x[r].y)),
                                     fmaxf(finite_abs(x[r].z), finite_abs(x[r].w))));
        }
    }
    const int e = max(block_exponent(warp_max(amax)), e_old);
    if (r0 > 0 && e > e_old) {
        for (int r = 0; r < kPageTokens; ++r) {
            if (r < r0 || r >= r0 + it.count) {
                uint32_t *p = reinterpret_cast<uint32_t *>(unit + code_offset(r, lane));
                *p = rescale_codes4(*p, e - e_old);
            }
        }
    }
    const float inv = pow2(-e);
#pragma unroll
    for (int r = 0; r < kPageTokens; ++r) {
        if (r < it.count) {
            *reinterpret_cast<uint32_t *>(unit + code_offset(r0 + r, lane)) = to_codes4(x[r], inv);
        }
    }
    if (lane == 0) {
        *exp_slot = e;
    }
}

template <typename T>
void launch_write_t(const PoolView &pool, const RopeView &rope, const BatchView &batch,
                    const WriteArgs &a, DeviceError *err, cudaStream_t stream) {
    const int64_t warps = static_cast<int64_t>(a.n_items) * (2 + (a.q != nullptr ? kGqa : 0)) * pool.n_head_kv;
    const unsigned blocks = static_cast<unsigned>((warps + kWriteWarps - 1) / kWriteWarps);
    if (pool.format == kCacheE4m3) {
        write_kernel<T, true><<<blocks, kWriteWarps * 32, 0, stream>>>(pool, rope, batch, a, err);
    } else {
        write_kernel<T, false><<<blocks, kWriteWarps * 32, 0, stream>>>(pool, rope, batch, a, err);
    }
}

// ======================================================================== read
// One CTA per page item; a thread takes 8 dims of one row and head at a time.
template <typename T, bool kE4m3>
__global__ void __launch_bounds__(256)
    read_kernel(PoolView pool, const RowItem *__restrict__ items, int layer, T *__restrict__ k_out,
                T *__restrict__ v_out, DeviceError *err) {
    const RowItem it = items[blockIdx.x];
    const int G = pool.n_head_kv;
    const int r0 = it.pos0 & 15;
    if (it.page < 0 || it.page >= pool.n_pages || it.count < 1 || r0 + it.count > kPageTokens) {
        if (threadIdx.x == 0) {
            record(err, kWhereRead, it.page, it.pos0);
        }
        return;
    }
    const int total = it.count * 2 * G * 16;
    for (int i = threadIdx.x; i < total; i += 256) {
        const int c = i & 15;  // 8 dims
        const int rest = i >> 4;
        const int head = rest % G;
        const int kv = (rest / G) & 1;
        const int r = rest / (2 * G);
        const int row = r0 + r;
        float4 lo, hi;
        if (kE4m3) {
            const uint8_t *unit =
                pool.base + code_unit_index(it.page, layer, head, pool.n_pages, G) * kCodeUnitBytes;
            const float scale = pow2(reinterpret_cast<const int *>(unit + 2 * kCodeBlockBytes)[kv]);
            const uint2 u = *reinterpret_cast<const uint2 *>(
                unit + kv * kCodeBlockBytes + row * kHeadDim + (((c >> 1) ^ (row & 7)) << 4) + (c & 1) * 8);
            lo = codes_to_float4(u.x);
            hi = codes_to_float4(u.y);
            lo = make_float4(lo.x * scale, lo.y * scale, lo.z * scale, lo.w * scale);
            hi = make_float4(hi.x * scale, hi.y * scale, hi.z * scale, hi.w * scale);
        } else {
            const uint8_t *block =
                pool.base + head_block_index(it.page, layer, kv, head, pool.n_pages, G) * kHeadBlockBytes;
            const __half *p =
                reinterpret_cast<const __half *>(block + row * kRowBytes + swizzled_chunk(row, c) * 16);
            const uint4 u = *reinterpret_cast<const uint4 *>(p);
            const __half2 *h = reinterpret_cast<const __half2 *>(&u);
            const float2 f0 = __half22float2(h[0]), f1 = __half22float2(h[1]);
            const float2 f2 = __half22float2(h[2]), f3 = __half22float2(h[3]);
            lo = make_float4(f0.x, f0.y, f1.x, f1.y);
            hi = make_float4(f2.x, f2.y, f3.x, f3.y);
        }
        T *dst = (kv != 0 ? v_out : k_out) +
                 (static_cast<int64_t>(it.row0 + r) * G + head) * kHeadDim + c * 8;
        store4(dst, lo);
        store4(dst + 4, hi);
    }
}

template <typename T>
void launch_read_t(const PoolView &pool, const RowItem *items, int32_t n_items, int layer, void *k_out,
                   void *v_out, DeviceError *err, cudaStream_t stream) {
    T *k = static_cast<T *>(k_out);
    T *v = static_cast<T *>(v_out);
    if (pool.format == kCacheE4m3) {
        read_kernel<T, true><<<n_items, 256, 0, stream>>>(pool, items, layer, k, v, err);
    } else {
        read_kernel<T, false><<<n_items, 256, 0, stream>>>(pool, items, layer, k, v, err);
    }
}

}  // namespace

void launch_write(const PoolView &pool, const RopeView &rope, const BatchView &batch,
                  const WriteArgs &args, DeviceError *err, cudaStream_t stream) {
    if (args.dtype == kDtypeF32) {
        launch_write_t<float>(pool, rope, batch, args, err, stream);
    } else if (args.dtype == kDtypeF16) {
        launch_write_t<__half>(pool, rope, batch, args, err, stream);
    } else {
        launch_write_t<__nv_bfloat16>(pool, rope, batch, args, err, stream);
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
