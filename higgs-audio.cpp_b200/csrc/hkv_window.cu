// hkv_window.cu -- attention of several new tokens per slot over the paged cache
// (prompts, refreshed windows): row i of a slot sees rows [0, used + i].
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "hkv_device.cuh"
#include "hkv_e4m3.cuh"
#include "hkv_internal.h"

namespace hkv {
namespace {

using namespace dev;

constexpr int kWhereWindow = 8;
constexpr int kDtypeF32 = 0;
constexpr int kDtypeF16 = 1;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_f32(float *p, float x) { *p = x; }
__device__ __forceinline__ void from_f32(__half *p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void from_f32(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }

// One CTA per (tile, KV head): 16 tokens x 4 query heads at a time, four threads
// a row (32 dims each), the pages of the cache through shared memory as F32.
template <typename T, bool kE4m3>
__global__ void __launch_bounds__(256)
    window_kernel(PoolView pool, const WindowTile *__restrict__ tiles, const int32_t *__restrict__ pages,
                  int layer, const T *__restrict__ q, int64_t q_stride, T *__restrict__ out, int64_t out_stride,
                  float scale_log2, DeviceError *err) {
    __shared__ float ks[kPageTokens][kHeadDim];
    __shared__ float vs[kPageTokens][kHeadDim];
    const WindowTile t = tiles[blockIdx.x];
    const int G = pool.n_head_kv;
    const int h = blockIdx.y;
    const int part = threadIdx.x & 3;
    const int head = (threadIdx.x >> 2) & 3;
    for (int sub = 0; sub < t.tokens; sub += 16) {
        const int tok = sub + (threadIdx.x >> 4);
        const bool live = tok < t.tokens;
        const int64_t row = t.row0 + (live ? tok : 0);
        const T *qp = q + row * q_stride + (kGqa * h + head) * kHeadDim + 32 * part;
        float qv[32], o[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            qv[i] = to_f32(qp[i]);
            o[i] = 0.f;
        }
        float m = -INFINITY, l = 0.f;
        const int last = t.pos0 + min(sub + 15, t.tokens - 1);  // last key any row of this pass sees
        const int mine = t.pos0 + tok;
        for (int p = 0; p * kPageTokens <= last; ++p) {
            __syncthreads();
            const int64_t page = pages[t.page_off + p];
            const bool ok = page >= 0 && page < pool.n_pages;
            if (!ok && threadIdx.x == 0 && atomicCAS(&err->code, 0, kErrBadIndex) == 0) {
                err->where = kWhereWindow;
                err->a = static_cast<int>(page);
                err->b = p;
            }
            for (int i = threadIdx.x; ok && i < 2 * kPageTokens * kHeadDim; i += 256) {
                const int kv = i / (kPageTokens * kHeadDim);
                const int r = (i / kHeadDim) % kPageTokens;
                const int d = i % kHeadDim;
                float x;
                if (kE4m3) {
                    const uint8_t *unit =
                        pool.base + code_unit_index(page, layer, h, pool.n_pages, G) * kCodeUnitBytes;
                    const float s = pow2(reinterpret_cast<const int *>(unit + 2 * kCodeBlockBytes)[kv]);
                    const uint32_t c = unit[kv * kCodeBlockBytes + r * kHeadDim + (((d >> 4) ^ (r & 7)) << 4) + (d & 15)];
                    x = codes_to_float4(c).x * s;
                } else {
                    const uint8_t *b =
                        pool.base + head_block_index(page, layer, kv, h, pool.n_pages, G) * kHeadBlockBytes;
                    x = __half2float(*reinterpret_cast<const __half *>(b + r * kRowBytes +
                                                                       swizzled_chunk(r, d >> 3) * 16 + (d & 7) * 2));
                }
                (kv ? vs : ks)[r][d] = x;
            }
            __syncthreads();
            for (int r = 0; r < kPageTokens && p * kPageTokens + r <= last; ++r) {
                float s = 0.f;
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    s += qv[i] * ks[r][32 * part + i];
                }
                s += __shfl_xor_sync(0xffffffffu, s, 1);
                s += __shfl_xor_sync(0xffffffffu, s, 2);
                if (p * kPageTokens + r <= mine) {
                    s *= scale_log2;
                    const float mn = fmaxf(m, s);
                    const float alpha = exp2f(m - mn);
                    const float w = exp2f(s - mn);
                    m = mn;
                    l = l * alpha + w;
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        o[i] = o[i] * alpha + w * vs[r][32 * part + i];
                    }
                }
            }
        }
        if (live) {
            T *op = out + row * out_stride + (kGqa * h + head) * kHeadDim + 32 * part;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                from_f32(op + i, o[i] / l);
            }
        }
        __syncthreads();
    }
}

template <typename T>
void launch_window_t(const PoolView &pool, const WindowArgs &a, DeviceError *err, cudaStream_t stream) {
    const dim3 grid(static_cast<unsigned>(a.n_tiles), static_cast<unsigned>(pool.n_head_kv));
    const T *q = static_cast<const T *>(a.q);
    T *out = static_cast<T *>(a.out);
    if (pool.format == kCacheE4m3) {
        window_kernel<T, true><<<grid, 256, 0, stream>>>(pool, a.tiles, a.pages, a.layer, q, a.q_stride, out,
                                                         a.out_stride, a.scale_log2, err);
    } else {
        window_kernel<T, false><<<grid, 256, 0, stream>>>(pool, a.tiles, a.pages, a.layer, q, a.q_stride, out,
                                                          a.out_stride, a.scale_log2, err);
    }
}

}  // namespace

void launch_window(const PoolView &pool, const WindowArgs &args, DeviceError *err, cudaStream_t stream) {
    if (args.dtype == kDtypeF32) {
        launch_window_t<float>(pool, args, err, stream);
    } else if (args.dtype == kDtypeF16) {
        launch_window_t<__half>(pool, args, err, stream);
    } else {
        launch_window_t<__nv_bfloat16>(pool, args, err, stream);
    }
}

}  // namespace hkv
