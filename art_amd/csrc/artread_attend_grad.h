// Gradient of the attention (include/artread.h).  Included by artread.hip only.
#pragma once
#include "artread_attend.h"

__device__ __forceinline__ float wave_max(float x) {
    for (int o = 32; o; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}
__device__ __forceinline__ float wave_sum(float x) {
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
    return x;
}
__device__ __forceinline__ int valid_of(const artread_attend_t& A, int64_t b, int64_t p) {
    if (!A.lengths) return (int)A.len;
    const int n = A.lengths[b * A.passages + p];
    return n < 0 ? 0 : (n < A.len ? n : (int)A.len);
}


// delta[b, h, t] = grad_out . out, and grad_q: one wave per query row
template <typename T>
__global__ __launch_bounds__(64) void attend_grad_q_simple_kernel(artread_attend_t A, artread_attend_grads_t G,
                                                                  float* __restrict__ delta) {
    __shared__ float qs[128], gs[128], ps[64];
    const int lane = threadIdx.x, dim = (int)A.dim;
    const int64_t total = A.batch * A.rows * A.heads;
    for (int64_t w = blockIdx.x; w < total; w += gridDim.x) {
        const int64_t h = w % A.heads, t = w / A.heads % A.rows, b = w / A.heads / A.rows;
        const int64_t kh = h / (A.heads / A.kv_heads);
        const T* q = (const T*)A.q + b * A.q_batch + t * A.q_row + h * A.q_head;
        const T* g = (const T*)G.grad_out + b * G.g_batch + t * G.g_row + h * G.g_head;
        const T* out = (const T*)A.out + w * dim;
        __syncthreads();
        float dl = 0.0f;
        for (int d = lane; d < 128; d += 64) {
            qs[d] = d < dim ? to_f32(q[d]) : 0.0f;
            gs[d] = d < dim ? to_f32(g[d]) : 0.0f;
            if (d < dim) dl += gs[d] * (to_f32(out[d]) + (A.rest ? to_f32(((const T*)A.rest + w * dim)[d]) : 0.0f));
        }
        dl = wave_sum(dl);
        const int64_t at = (b * A.heads + h) * A.rows + t;
        if (lane == 0) delta[at] = dl;
        const float lse = A.lse[at];
        __syncthreads();
        float o0 = 0.0f, o1 = 0.0f;
        for (int64_t p = 0; p < A.passages; ++p) {
            const int n = valid_of(A, b, p);
            const T* k = (const T*)A.k + b * A.k_batch + p * A.k_passage + kh * A.k_head;
            const T* v = (const T*)A.v + b * A.v_batch + p * A.v_passage + kh * A.v_head;
            for (int j0 = 0; j0 < n; j0 += 64) {
                float ds = 0.0f;
                if (j0 + lane < n) {
                    float s = 0.0f, dp = 0.0f;
                    for (int d = 0; d < dim; ++d) {
                        s += qs[d] * to_f32(k[(int64_t)(j0 + lane) * A.k_row + d]);
                        dp += gs[d] * to_f32(v[(int64_t)(j0 + lane) * A.v_row + d]);
                    }
                    ds = exp2f((s * A.scale - lse) * kLog2e) * (dp - dl);
                }
                __syncthreads();
                ps[lane] = ds;
                __syncthreads();
                const int c = n - j0 < 64 ? n - j0 : 64;
                for (int j = 0; j < c; ++j) {
                    const T* kr = k + (int64_t)(j0 + j) * A.k_row;
                    if (lane < dim) o0 += ps[j] * to_f32(kr[lane]);
                    if (lane + 64 < dim) o1 += ps[j] * to_f32(kr[lane + 64]);
                }
            }
        }
        T* gq = (T*)G.grad_q + w * dim;
        if (lane < dim) gq[lane] = from_f32<T>(o0 * A.scale);
        if (lane + 64 < dim) gq[lane + 64] = from_f32<T>(o1 * A.scale);
    }
}

// grad_k and grad_v: one wave per key (b, p, j, kh) over all rows of the heads that share it
template <typename T>
__global__ __launch_bounds__(64) void attend_grad_kv_simple_kernel(artread_attend_t A, artread_attend_grads_t G,
                                                                   const float* __restrict__ delta) {
    __shared__ float ks[128], vs[128], ps[64], es[64];
    const int lane = threadIdx.x, dim = (int)A.dim;
    const int64_t share = A.heads / A.kv_heads, rows = A.rows * share;
    const int64_t total = A.batch * A.passages * A.len * A.kv_heads;
    for (int64_t w = blockIdx.x; w < total; w += gridDim.x) {
        const int64_t kh = w % A.kv_heads, j = w / A.kv_heads % A.len, p = w / A.kv_heads / A.len % A.passages;
        const int64_t b = w / A.kv_heads / A.len / A.passages;
        T* gk = (T*)G.grad_k + w * dim;
        T* gv = (T*)G.grad_v + w * dim;
        float k0 = 0.0f, k1 = 0.0f, v0 = 0.0f, v1 = 0.0f;
        if (j < valid_of(A, b, p)) {
            const T* k = (const T*)A.k + b * A.k_batch + p * A.k_passage + j * A.k_row + kh * A.k_head;
            const T* v = (const T*)A.v + b * A.v_batch + p * A.v_passage + j * A.v_row + kh * A.v_head;
            __syncthreads();
            for (int d = lane; d < 128; d += 64) {
                ks[d] = d < dim ? to_f32(k[d]) : 0.0f;
                vs[d] = d < dim ? to_f32(v[d]) : 0.0f;
            }
            __syncthreads();
            for (int64_t r0 = 0; r0 < rows; r0 += 64) {
                float e = 0.0f, ds = 0.0f;
                const int64_t r = r0 + lane;
                if (r < rows) {
                    const int64_t t = r / share, h = kh * share + r % share;
                    const T* q = (const T*)A.q + b * A.q_batch + t * A.q_row + h * A.q_head;
                    const T* g = (const T*)G.grad_out + b * G.g_batch + t * G.g_row + h * G.g_head;
                    float s = 0.0f, dp = 0.0f;
                    for (int d = 0; d < dim; ++d) {
                        s += ks[d] * to_f32(q[d]);
                        dp += vs[d] * to_f32(g[d]);
                    }
                    const int64_t at = (b * A.heads + h) * A.rows + t;
                    e = exp2f((s * A.scale - A.lse[at]) * kLog2e);
                    ds = e * (dp - delta[at]);
                }
                __syncthreads();
                ps[lane] = e;
                es[lane] = ds;
                __syncthreads();
                const int c = rows - r0 < 64 ? (int)(rows - r0) : 64;
                for (int i = 0; i < c; ++i) {
                    const int64_t t = (r0 + i) / share, h = kh * share + (r0 + i) % share;
                    const T* q = (const T*)A.q + b * A.q_batch + t * A.q_row + h * A.q_head;
                    const T* g = (const T*)G.grad_out + b * G.g_batch + t * G.g_row + h * G.g_head;
                    if (lane < dim) {
                        k0 += es[i] * to_f32(q[lane]);
                        v0 += ps[i] * to_f32(g[lane]);
                    }
                    if (lane + 64 < dim) {
                        k1 += es[i] * to_f32(q[lane + 64]);
                        v1 += ps[i] * to_f32(g[lane + 64]);
                    }
                }
            }
        }
        if (lane < dim) {
            gk[lane] = from_f32<T>(k0 * A.scale);
            gv[lane] = from_f32<T>(v0);
        }
        if (lane + 64 < dim) {
            gk[lane + 64] = from_f32<T>(k1 * A.scale);
            gv[lane + 64] = from_f32<T>(v1);
        }
    }
}
