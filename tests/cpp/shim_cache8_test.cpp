// include/hkv_pipeline.hpp with an 8-bit cache, and window_layer: on a host-only engine
// (no GPU) the type and the refusals; with an argument "gpu", prompt rows through
// window_layer against the one-token steps of decode_layer on the GPU.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdio>
#include <cstring>
#include <stdexcept>

#include "hkv_pipeline.hpp"

#define EXPECT(c)                                                        \
    do {                                                                 \
        if (!(c)) {                                                      \
            std::fprintf(stderr, "FAILED %s:%d: %s\n", __FILE__, __LINE__, #c); \
            return 1;                                                    \
        }                                                                \
    } while (0)

static int host_only() {
    hkv_config cfg;
    hkv_config_default(&cfg);
    cfg.n_layers = 1;
    cfg.n_pages = 8;
    cfg.max_slots = 2;
    cfg.context_length = 128;
    cfg.device = -1;
    int32_t type = -1;
    hkv_pipeline::PagedKvRuntime f16(cfg), rt(cfg, HKV_CACHE_E4M3);
    EXPECT(hkv_engine_cache_type(f16.engine(), &type) == HKV_OK && type == HKV_CACHE_F16);
    EXPECT(hkv_engine_cache_type(rt.engine(), &type) == HKV_OK && type == HKV_CACHE_E4M3);
    auto s = hkv_pipeline::acquire_backend_kv_cache_slot(rt, 32);
    bool refused = false;
    try {
        hkv_pipeline::window_layer(rt, 0, {s.slot()}, {1, 2}, nullptr, nullptr, nullptr, nullptr, nullptr);
    } catch (const std::out_of_range &) {
        refused = true;
    }
    EXPECT(refused);
    refused = false;
    try {
        hkv_pipeline::window_layer(rt, 0, {s.slot()}, {1}, nullptr, nullptr, nullptr, nullptr, nullptr);
    } catch (const std::runtime_error &) {
        refused = true;
    }
    EXPECT(refused);
    return 0;
}

static int on_gpu() {
    const int T = 40, HQ = 32, G = 8, D = 128;
    hkv_config cfg;
    hkv_config_default(&cfg);
    cfg.n_layers = 1;
    cfg.n_pages = 8;
    cfg.max_slots = 2;
    cfg.context_length = 128;
    hkv_pipeline::PagedKvRuntime rt(cfg);  // F16: a row's cache bits do not hang on later rows
    auto a = hkv_pipeline::acquire_backend_kv_cache_slot(rt, T), b = hkv_pipeline::acquire_backend_kv_cache_slot(rt, T);
    std::vector<float> q(T * HQ * D), k(T * G * D), v(T * G * D), o1(q.size()), o2(q.size());
    uint32_t x = 1;
    auto next = [&]() {
        x = x * 1664525u + 1013904223u;
        return static_cast<float>(static_cast<int32_t>(x)) * 4.6566129e-10f;
    };
    for (auto *p : {&q, &k, &v}) {
        for (float &y : *p) {
            y = next();
        }
    }
    float *dq, *dk, *dv, *out;
    EXPECT(cudaMalloc(&dq, q.size() * 4) == cudaSuccess && cudaMalloc(&dk, k.size() * 4) == cudaSuccess &&
           cudaMalloc(&dv, v.size() * 4) == cudaSuccess && cudaMalloc(&out, q.size() * 4) == cudaSuccess);
    auto up = [](float *d, const std::vector<float> &h) {
        return cudaMemcpy(d, h.data(), h.size() * 4, cudaMemcpyHostToDevice) == cudaSuccess;
    };
    EXPECT(up(dq, q) && up(dk, k) && up(dv, v));
    for (int t = 0; t < T; ++t) {
        hkv_pipeline::decode_layer(rt, 0, {a.slot()}, dq + t * HQ * D, dk + t * G * D, dv + t * G * D, out + t * HQ * D,
                                   nullptr);
        a.advance(1);
    }
    hkv_pipeline::check(rt.engine(), hkv_sync_check(rt.engine(), nullptr), "sync");
    EXPECT(cudaMemcpy(o1.data(), out, o1.size() * 4, cudaMemcpyDeviceToHost) == cudaSuccess);
    hkv_pipeline::window_layer(rt, 0, {b.slot()}, {T}, dq, dk, dv, out, nullptr);
    b.advance(T);
    hkv_pipeline::check(rt.engine(), hkv_sync_check(rt.engine(), nullptr), "sync");
    EXPECT(cudaMemcpy(o2.data(), out, o2.size() * 4, cudaMemcpyDeviceToHost) == cudaSuccess);
    // K and V in the cache are the same bits on both sides.  |q| and |k| are at most sqrt(2)
    // after their rotation, so the sizes of a logit's products add up to at most
    // S = 256 / sqrt(128) = 22.7; q in two F16 parts is off by 2^-22 of S at most and 16 cut
    // steps of the sum by 2^-23 of it each: 22.7 (2^-22 + 2^-19) = 4.9e-5, which is a
    // weight's relative error, and with the sum's at most twice that of an output (|v| < 1).
    // One block's 16 cut steps of the output add 2^-19, exp2 2^-21: 1.1e-4 on each side.
    for (size_t i = 0; i < o1.size(); ++i) {
        EXPECT(std::fabs(o1[i] - o2[i]) < 2.2e-4f);
    }
    cudaFree(dq);
    cudaFree(dk);
    cudaFree(dv);
    cudaFree(out);
    return 0;
}

int main(int argc, char **argv) {
    const int rc = argc > 1 && std::strcmp(argv[1], "gpu") == 0 ? on_gpu() : host_only();
    if (rc == 0) {
        std::puts("shim cache8 ok");
    }
    return rc;
}
