// Element access to the page pool in any of its formats, for the coverage kernels.
#pragma once
#include "common.cuh"

namespace emlx {

constexpr int kMaxHeadDim = 256;
constexpr int kPerLane = kMaxHeadDim / 32;

struct PoolView {
    emlx_pool p;
    __device__ __forceinline__ float key(int64_t page, int off, int h, int d) const {
        const int D = p.head_dim, Hkv = p.num_kv_heads, bs = p.block_size;
        if (p.kv_format == EMLX_KV_FLOAT) {
            const int64_t i = ((page * bs + off) * Hkv + h) * D + d;
            if (p.kv_dtype == EMLX_F16) return __half2float(((const __half*)p.key_cache)[i]);
            if (p.kv_dtype == EMLX_BF16) return __bfloat162float(((const __nv_bfloat16*)p.key_cache)[i]);
            return ((const float*)p.key_cache)[i];
        }
        const int bits = p.kv_format;
        const uint8_t* row = (const uint8_t*)p.key_cache + ((page * bs + off) * Hkv + h) * (int64_t)(D * bits / 8);
        const int code = bits == 8 ? row[d] : ((row[d >> 1] >> ((d & 1) * 4)) & 0xF);
        const int64_t sb = ((page * Hkv + h) * bs + off) * (D / kQuantGroup) + d / kQuantGroup;
        return __fadd_rn(__fmul_rn(__half2float(((const __half*)p.k_scale)[sb]), (float)code),
                         __half2float(((const __half*)p.k_bias)[sb]));
    }
    __device__ __forceinline__ float value(int64_t page, int off, int h, int d) const {
        const int D = p.head_dim, Hkv = p.num_kv_heads, bs = p.block_size;
        if (p.kv_format == EMLX_KV_FLOAT) {
            const int64_t i = ((page * bs + off) * Hkv + h) * D + d;
            if (p.kv_dtype == EMLX_F16) return __half2float(((const __half*)p.value_cache)[i]);
            if (p.kv_dtype == EMLX_BF16) return __bfloat162float(((const __nv_bfloat16*)p.value_cache)[i]);
            return ((const float*)p.value_cache)[i];
        }
        const int bits = p.kv_format;
        const uint8_t* col = (const uint8_t*)p.value_cache + ((page * Hkv + h) * D + d) * (int64_t)(bs * bits / 8);
        const int code = bits == 8 ? col[off] : ((col[off >> 1] >> ((off & 1) * 4)) & 0xF);
        const int64_t sb = ((page * Hkv + h) * bs + off) * (D / kQuantGroup) + d / kQuantGroup;
        return __fadd_rn(__fmul_rn(__half2float(((const __half*)p.v_scale)[sb]), (float)code),
                         __half2float(((const __half*)p.v_bias)[sb]));
    }
};

}  // namespace emlx
