// serve.h -- batched serving operators: the paged 8-bit KV cache (kv8.cu, kv8_attn.cu), attention
// over packed prompts (attn_packed.cu) and log probabilities (logprobs.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "common.cuh"

namespace tptc {

// Eight consecutive elements of a row, as loaded and as f32, whatever the element type.
template <typename T>
struct Raw8 {
    uint4 w[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Raw8<T> load_raw8(const T* p) {
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) r.w[i] = reinterpret_cast<const uint4*>(p)[i];
    return r;
}
template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T>& v, float (&x)[8]) {
    const uint32_t* r = reinterpret_cast<const uint32_t*>(&v);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = __uint_as_float(r[i]);
    } else if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(reinterpret_cast<const __half2&>(r[i]));
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            x[2 * i] = __uint_as_float(r[i] << 16), x[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
    }
}
// Two f32 as a pair of T in one word (round to nearest), the first in the low half.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]),
                                                  pack2<T>(x[6], x[7]));
    }
}

template <typename T>
__device__ __forceinline__ float to_f32(T x) {
    return static_cast<float>(x);
}

// kv8.cu
struct Kv8Append {
    tptc_kv8 c;
    tptc_rope rope;  // dim 0: no rotation
    const void *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;
    int n_heads;  // 0: no queries
    void *q_out, *k_out;
    const int32_t *cu, *start;
    int n_tokens, max_new;
    int units;  // pages that a sequence can touch, 0: units are counted on the device (filled by the launcher)
};
cudaError_t launch_kv8_append(int type, Kv8Append p, cudaStream_t st);

struct Kv8Read {
    tptc_kv8 c;
    const int32_t *cu, *start;
    int n_tokens, max_rows;
    void *k_out, *v_out;
    int units, heads_per_cta;  // units as above; filled by the launcher
};
cudaError_t launch_kv8_read(int type, Kv8Read p, cudaStream_t st);

// kv8_attn.cu
struct Kv8Attn {
    tptc_kv8 c;
    const void* q;
    int64_t q_stride;
    const int32_t* len;
    int n_heads;
    void* out;
    uint8_t* workspace;  // kv8_attn_workspace() bytes; the counters at its end are zero between calls
};
bool kv8_attn_fits(const tptc_kv8& c);  // whether the kernel's sums hold the longest batch that the table allows
size_t kv8_attn_workspace(const tptc_kv8& c, int n_heads, int sms);
cudaError_t launch_kv8_attn(int type, const Kv8Attn& a, int sms, cudaStream_t st);
cudaError_t kv8_attn_init_device();

// attn_packed.cu
struct AttnPacked {
    const void *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;
    void* out;
    const int32_t *cu_q, *cu_k;
    int n_seq, n_q, n_k, max_q, n_heads, n_kv, head_dim;
    int32_t* status;
};
cudaError_t launch_attn_packed(int type, const AttnPacked& a, cudaStream_t st);
cudaError_t attn_packed_init_device();

// logprobs.cu
constexpr int kMaxTop = 32;
struct LogprobParams {
    const void* logits;
    int rows, vocab;
    int64_t row_stride;
    const int32_t* token;
    float *logprob, *entropy;
    int n_top;
    int32_t* top_id;
    float* top_logprob;
};
cudaError_t launch_logprobs(int type, const LogprobParams& p, int sms, cudaStream_t st);
cudaError_t logprobs_init_device();

// Attributes of this group's kernels on the current device (kv8.cu).
cudaError_t serve_init_device();

}  // namespace tptc
