// Gradient of the attention (include/artread.h).  Included by artread.hip only.
//
// With P = exp(scale * S - lse) and dP = dO V^T:  dS = P (dP - delta), delta = rowsum(dO * O),
//   dV = P^T dO,  dQ = scale dS K,  dK = scale dS^T Q.
// Two walks, each computing S and dP anew (two extra products instead of atomics or a pass over stored scores):
// the row walk keeps its rows of dQ and goes over the keys as the forward does, the key walk keeps its keys of dK
// and dV and goes over the rows, those of the heads that share a key head among them.  In both a lane owns one
// column of S (a row, or a key), so P and dS are already the B operands of the second products.
#pragma once
#include "artread_attend.h"

// log-sum and delta of every row in the order (batch entry, key head, r), the log-sum in powers of two and with the
// factor that f16 weights carry: P = exp2(S * c - x)
struct RowStat {
    float x, delta;
};

// 16 lanes per row, eight columns each
template <typename T>
__global__ __launch_bounds__(256) void attend_delta_kernel(artread_attend_t A, artread_attend_grads_t G, AttendPlan P,
                                                           int64_t all_rows, RowStat* __restrict__ stats) {
    const int lane = threadIdx.x & 15, d = lane * 8;
    for (int64_t R = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); R < all_rows; R += (int64_t)gridDim.x * 16) {
        const int64_t r = R % P.row_count, bk = R / P.row_count, kh = bk % A.kv_heads, b = bk / A.kv_heads;
        const int64_t t = r / P.share, h = kh * P.share + r % P.share;
        const int64_t at = ((b * A.rows + t) * A.heads + h) * A.dim + d;
        float sum = 0.0f;
        if (d < (int)A.dim) {
            const Vec<T, 8> g = load_vec<T, 8>((const T*)G.grad_out + b * G.g_batch + t * G.g_row + h * G.g_head + d);
            const Vec<T, 8> o = load_vec<T, 8>((const T*)A.out + at);
            Vec<T, 8> e = {};
            if (A.rest) e = load_vec<T, 8>((const T*)A.rest + at);
#pragma unroll
            for (int x = 0; x < 8; ++x) sum += (float)g.x[x] * ((float)o.x[x] + (float)e.x[x]);
        }
#pragma unroll
        for (int x = 8; x; x >>= 1) sum += __shfl_xor(sum, x);
        if (lane == 0) {
            const float lse = A.lse[(b * A.heads + h) * A.rows + t];
            // a row without keys has no weight anywhere
            stats[R] = RowStat{lse == -INFINITY ? INFINITY : lse * kLog2e - Mma<T>::kWeightLog2, sum};
        }
    }
}

// dS of f16 spans more than f16 does (a loss of 1e-6, or one scaled by thousands): each column keeps a power of two
// beside it, chosen when the first value that is not zero arrives and lowered when a value outgrows it; the
// accumulators follow.  bf16 has the exponents of f32 and needs none.
template <typename T>
struct Spread {
    float f = 1.0f;
    __device__ __forceinline__ float inverse() const { return 1.0f; }
    template <int N>
    __device__ __forceinline__ void fit(f32x16&, f32x16 (&)[N]) {}
};
template <>
struct Spread<f16> {
    float f = 1.0f, most = 0.0f;   // f * most is 2^14
    __device__ __forceinline__ float inverse() const { return 1.0f / f; }
    template <int N>
    __device__ __forceinline__ void fit(f32x16& ds, f32x16 (&acc)[N]) {
        float top = fabsf(ds[0]);
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, fabsf(ds[i]));
        if (__any(top > most)) {
            top = fmaxf(top, other_half(top));
            if (top > most) {
                int e = 10 - ilogbf(top);                       // top * 2^e is in [2^10, 2^11)
                e = e < -100 ? -100 : (e > 100 ? 100 : e);
                const float g = ldexpf(1.0f, e), change = most == 0.0f ? 0.0f : g / f;
                f = g;
                most = ldexpf(1.0f, 14 - e);
#pragma unroll
                for (int x = 0; x < N; ++x)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[x][i] *= change;
            }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) ds[i] *= f;
    }
};

template <typename T>
__device__ __forceinline__ void put4(T* p, const float* x) {
    Vec<T, 4> w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w.x[e] = (T)x[e];
    store_vec<T, 4>(p, w);
}

// ---- dQ: the row walk -----------------------------------------------------------------------------------
// NW waves of 32 rows share tiles of 32 * KB keys, double-buffered in LDS.  With P.splits > 1 each split leaves
// its f32 part of dQ at part + split * (all of dQ).
template <typename T, int DP, int NW, int KB>
__global__ __launch_bounds__(64 * NW, DP == 64 ? 2 : 1) void attend_grad_q_kernel(artread_attend_t A, artread_attend_grads_t G,
                                                                    AttendPlan P, const RowStat* __restrict__ stats,
                                                                    float* __restrict__ part) {
    __shared__ __attribute__((aligned(16))) T ktile[2][32 * KB * DP];
    __shared__ __attribute__((aligned(16))) T vtile[2][32 * KB * DP];
    typedef typename Mma<T>::V8 V8;
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = uniform(threadIdx.x >> 6);
    const int dim = (int)A.dim;
    const int64_t total = P.items * P.splits;
    for (int64_t id = blockIdx.x; id < (total + 7) / 8 * 8; id += gridDim.x) {
        const int64_t w = xcd_item(id, total);
        if (w >= total) continue;
        const int64_t rb = w % P.row_blocks, other = w / P.row_blocks;
        const int split = (int)(other % P.splits);
        const int64_t bk = other / P.splits, kh = bk % A.kv_heads, b = bk / A.kv_heads;
        const int64_t r = (rb * NW + wave) * 32 + (lane & 31);
        V8 q[DP / 16], g[DP / 16];
        load_q<T, DP>(A, P, (const T*)A.q, A.q_batch, A.q_row, A.q_head, b, kh, r, half, P.q_and, P.q_xor, q);
        load_q<T, DP>(A, P, (const T*)G.grad_out, G.g_batch, G.g_row, G.g_head, b, kh, r, half, 0xffffffffu, 0u, g);
        RowStat st{INFINITY, 0.0f};
        if (r < P.row_count) st = stats[bk * P.row_count + r];
        f32x16 acc[DP / 32];
        Spread<T> spread;
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) acc[db] = f32x16{};
        constexpr int CH = DP / 8, TR = 64 * NW / CH, TN = 32 * KB / TR;
        const int trow = threadIdx.x / CH, tchunk = threadIdx.x % CH;
        const T* kbase = (const T*)A.k + b * A.k_batch + kh * A.k_head + (int64_t)trow * A.k_row + 8 * tchunk;
        const T* vbase = (const T*)A.v + b * A.v_batch + kh * A.v_head + (int64_t)trow * A.v_row + 8 * tchunk;
        V8 kr[TN], vr[TN];
        Walk<32 * KB> walk;
        walk.start(A, b, split, P.splits);
        auto load = [&]() {
            const int left = walk.n - walk.j0;
            const T* kp = kbase + walk.p * A.k_passage + walk.j0 * A.k_row;
            const T* vp = vbase + walk.p * A.v_passage + walk.j0 * A.v_row;
#pragma unroll
            for (int x = 0; x < TN; ++x) {
                const bool ok = trow + x * TR < left && 8 * tchunk < dim;
                kr[x] = load8<T>(kp + (int64_t)x * TR * A.k_row, ok);
                vr[x] = load8<T>(vp + (int64_t)x * TR * A.v_row, ok);
            }
        };
        auto put = [&](int buf) {
#pragma unroll
            for (int x = 0; x < TN; ++x) {
                const int row = trow + x * TR;
                *(V8*)(ktile[buf] + row * DP + tile_chunk<DP>(row, tchunk) * 8) = kr[x];
                *(V8*)(vtile[buf] + row * DP + tile_chunk<DP>(row, tchunk) * 8) = vr[x];
            }
        };
        bool more = walk.settle();
        if (more) {
            load();
            put(0);
        }
        __syncthreads();
        int buf = 0;
        while (more) {
            const int left = walk.n - walk.j0;
            walk.advance();
            more = walk.settle();
            if (more) load();
            const T* kt = ktile[buf];
            const T* vt = vtile[buf];
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
                for (int k = 0; k < DP / 16; ++k) {
                    s = Mma<T>::mul(lds_rows<T, DP>(kt, 32 * kb + (lane & 31), k, half), q[k], s);
                    dp = Mma<T>::mul(lds_rows<T, DP>(vt, 32 * kb + (lane & 31), k, half), g[k], dp);
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], P.c, -st.x)) * (dp[i] - st.delta);
                if (left < 32 * KB) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (32 * kb + 8 * (i >> 2) + 4 * half + (i & 3) >= left) s[i] = 0.0f;
                }
                spread.fit(s, acc);
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
                    const V8 ds = weights8<T>(s, ks);
#pragma unroll
                    for (int db = 0; db < DP / 32; ++db)
                        acc[db] = Mma<T>::mul(lds_columns<T, DP>(kt, 32 * kb + 16 * ks, db, lane), ds, acc[db]);
                }
            }
            if (more) put(buf ^ 1);
            __syncthreads();
            buf ^= 1;
        }
        if (r < P.row_count) {
            const int64_t t = r / P.share, h = kh * P.share + r % P.share;
            const int64_t at = ((b * A.rows + t) * A.heads + h) * dim;
            const float f = A.scale * spread.inverse() * P.unweight;
#pragma unroll
            for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int d = 32 * db + 8 * x + 4 * half;
                    const float y[4] = {f * acc[db][4 * x], f * acc[db][4 * x + 1], f * acc[db][4 * x + 2], f * acc[db][4 * x + 3]};
                    if (d >= dim) continue;
                    if (P.splits > 1) *(float4*)(part + split * (A.batch * A.rows * A.heads * dim) + at + d) = make_float4(y[0], y[1], y[2], y[3]);
                    else put4<T>((T*)G.grad_q + at + d, y);
                }
        }
    }
}

// ---- dK and dV: the key walk ------------------------------------------------------------------------------
// Four waves of 32 keys of one passage share tiles of 32 rows of Q and dO, double-buffered in LDS: each is read as
// rows for S and dP and transposed for dK and dV.  With P.splits > 1 the rows are dealt to splits, which leave f32
// parts of dK and dV.
template <typename T, int DP>
__global__ __launch_bounds__(256, DP == 64 ? 2 : 1) void attend_grad_kv_kernel(artread_attend_t A, artread_attend_grads_t G,
                                                                  AttendPlan P, const RowStat* __restrict__ stats,
                                                                  float* __restrict__ part) {
    __shared__ __attribute__((aligned(16))) T qtile[2][32 * DP];
    __shared__ __attribute__((aligned(16))) T gtile[2][32 * DP];
    __shared__ __attribute__((aligned(16))) RowStat stile[2][32];
    typedef typename Mma<T>::V8 V8;
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = uniform(threadIdx.x >> 6);
    const int dim = (int)A.dim;
    const int64_t key_blocks = (A.len + 127) / 128;
    const int64_t total = P.items * P.splits;   // batch x passages x key_blocks x kv_heads x splits
    for (int64_t w = blockIdx.x; w < total; w += gridDim.x) {
        const int split = (int)(w % P.splits);
        int64_t item = w / P.splits;
        const int64_t kh = item % A.kv_heads;
        item /= A.kv_heads;
        const int64_t j0 = item % key_blocks * 128;
        item /= key_blocks;
        const int64_t p = item % A.passages, b = item / A.passages;
        int n = (int)A.len;
        if (A.lengths) {
            const int x = uniform(A.lengths[b * A.passages + p]);
            n = x < n ? x : n;
        }
        const int64_t j = j0 + 32 * wave + (lane & 31);
        f32x16 dk[DP / 32], dv[DP / 32];
        Spread<T> spread;
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) dk[db] = dv[db] = f32x16{};
        if (j0 < n) {   // uniform over the workgroup
            V8 kf[DP / 16], vf[DP / 16];
            const T* kp = (const T*)A.k + b * A.k_batch + p * A.k_passage + j * A.k_row + kh * A.k_head + 8 * half;
            const T* vp = (const T*)A.v + b * A.v_batch + p * A.v_passage + j * A.v_row + kh * A.v_head + 8 * half;
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) {
                const bool ok = j < n && 16 * s + 8 * half < dim;
                union {
                    V8 v;
                    uint32_t u[4];
                } x;
                x.v = load8<T>(kp + 16 * s, ok);
#pragma unroll
                for (int e = 0; e < 4; ++e) x.u[e] = (x.u[e] & P.q_and) ^ P.q_xor;   // scale's sign, on this side of S
                kf[s] = x.v;
                vf[s] = load8<T>(vp + 16 * s, ok);
            }
            constexpr int CH = DP / 8, TR = 256 / CH, TN = 32 / TR;   // threads per row, rows side by side, steps
            const int trow = threadIdx.x / CH, tchunk = threadIdx.x % CH;
            V8 qr[TN], gr[TN];
            RowStat sr;
            const int64_t tiles = (P.row_count + 31) / 32;
            auto load = [&](int64_t tile) {
#pragma unroll
                for (int x = 0; x < TN; ++x) {
                    const int64_t r = tile * 32 + trow + x * TR;
                    const int64_t t = r / P.share, h = kh * P.share + r % P.share;
                    const bool ok = r < P.row_count && 8 * tchunk < dim;
                    qr[x] = load8<T>((const T*)A.q + b * A.q_batch + t * A.q_row + h * A.q_head + 8 * tchunk, ok);
                    gr[x] = load8<T>((const T*)G.grad_out + b * G.g_batch + t * G.g_row + h * G.g_head + 8 * tchunk, ok);
                }
                const int64_t r = tile * 32 + threadIdx.x;
                sr = RowStat{INFINITY, 0.0f};   // rows that are not there have no weight
                if (threadIdx.x < 32 && r < P.row_count) sr = stats[(b * A.kv_heads + kh) * P.row_count + r];
            };
            auto put = [&](int buf) {
#pragma unroll
                for (int x = 0; x < TN; ++x) {
                    const int row = trow + x * TR;
                    *(V8*)(qtile[buf] + row * DP + tile_chunk<DP>(row, tchunk) * 8) = qr[x];
                    *(V8*)(gtile[buf] + row * DP + tile_chunk<DP>(row, tchunk) * 8) = gr[x];
                }
                if (threadIdx.x < 32) stile[buf][threadIdx.x] = sr;
            };
            if (split < tiles) {
                load(split);
                put(0);
            }
            __syncthreads();
            int buf = 0;
            for (int64_t tile = split; tile < tiles; tile += P.splits) {
                const bool more = tile + P.splits < tiles;
                if (more) load(tile + P.splits);
                if (j0 + 32 * wave < n) {   // uniform over the wave
                    const T* qt = qtile[buf];
                    const T* gt = gtile[buf];
                    f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k) {
                        s = Mma<T>::mul(lds_rows<T, DP>(qt, lane & 31, k, half), kf[k], s);
                        dp = Mma<T>::mul(lds_rows<T, DP>(gt, lane & 31, k, half), vf[k], dp);
                    }
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const float4 a = *(const float4*)&stile[buf][8 * x + 4 * half];
                        const float4 c = *(const float4*)&stile[buf][8 * x + 4 * half + 2];
                        const float xs[4] = {a.x, a.z, c.x, c.z}, ds[4] = {a.y, a.w, c.y, c.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int i = 4 * x + e;
                            s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], P.c, -xs[e]));
                            dp[i] = s[i] * (dp[i] - ds[e]);
                        }
                    }
                    spread.fit(dp, dk);
#pragma unroll
                    for (int ks = 0; ks < 2; ++ks) {
                        const V8 pw = weights8<T>(s, ks), ds = weights8<T>(dp, ks);
#pragma unroll
                        for (int db = 0; db < DP / 32; ++db) {
                            dv[db] = Mma<T>::mul(lds_columns<T, DP>(gt, 16 * ks, db, lane), pw, dv[db]);
                            dk[db] = Mma<T>::mul(lds_columns<T, DP>(qt, 16 * ks, db, lane), ds, dk[db]);
                        }
                    }
                }
                if (more) put(buf ^ 1);
                __syncthreads();
                buf ^= 1;
            }
        }
        if (j < A.len) {
            const int64_t at = (((b * A.passages + p) * A.len + j) * A.kv_heads + kh) * dim;
            const int64_t all = A.batch * A.passages * A.len * A.kv_heads * dim;
            const float fv = P.unweight, fk = A.scale * spread.inverse() * P.unweight;
#pragma unroll
            for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int d = 32 * db + 8 * x + 4 * half;
                    if (d >= dim) continue;
                    float yk[4], yv[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {   // behind the length: zeros, whatever the accumulators hold
                        yk[e] = j < n ? fk * dk[db][4 * x + e] : 0.0f;
                        yv[e] = j < n ? fv * dv[db][4 * x + e] : 0.0f;
                    }
                    if (P.splits > 1) {
                        *(float4*)(part + split * 2 * all + at + d) = make_float4(yk[0], yk[1], yk[2], yk[3]);
                        *(float4*)(part + (split * 2 + 1) * all + at + d) = make_float4(yv[0], yv[1], yv[2], yv[3]);
                    } else {
                        put4<T>((T*)G.grad_k + at + d, yk);
                        put4<T>((T*)G.grad_v + at + d, yv);
                    }
                }
        }
    }
}

// out = sum of `splits` f32 parts `stride` apart, in order, rounded once; n is a multiple of 8
template <typename T>
__global__ __launch_bounds__(256) void attend_sum_kernel(const float* __restrict__ part, int64_t stride, int splits,
                                                         T* __restrict__ out, int64_t n) {
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += (int64_t)gridDim.x * 1024) {
        float y[4] = {0, 0, 0, 0};
#pragma unroll 4
        for (int s = 0; s < splits; ++s) {
            const float4 x = *(const float4*)(part + s * stride + i);
            y[0] += x.x;
            y[1] += x.y;
            y[2] += x.z;
            y[3] += x.w;
        }
        put4<T>(out + i, y);
    }
}
