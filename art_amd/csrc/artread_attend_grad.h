// Gradient of the attention (include/artread.h).  Included by artread.hip only.
//
// With P = exp(scale * S - lse) and dP = dO V^T:  dS = P (dP - delta), delta = rowsum(dO * O),
//   dV = P^T dO,  dQ = scale dS K,  dK = scale dS^T Q.
// Two walks, each computing S and dP anew (two extra products instead of atomics or a pass over stored scores):
// the row walk keeps its rows of dQ and goes over the keys as the forward does, the key walk keeps its keys of dK
// and dV and goes over the rows, those of the heads that share a key head among them.  In both a lane owns one
// column of S (a row, or a key), so P and dS are already the B operands of the second products.
#pragma once
#include <type_traits>

#include "artread_attend.h"

// log-sum and delta of every row in the order (batch entry, key head, r), the log-sum in powers of two and with the
// factor that f16 weights carry: P = exp2(S * c - x)
struct RowStat {
    float x, delta;
};

// 16 lanes per row, eight columns each.  The rows of a key head are padded to whole tiles of 32.
template <typename T>
__global__ __launch_bounds__(256) void attend_delta_kernel(artread_attend_t A, artread_attend_grads_t G, AttendPlan P,
                                                           int64_t all_rows, RowStat* __restrict__ stats) {
    const int lane = threadIdx.x & 15, d = lane * 8;
    for (int64_t R = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); R < all_rows; R += (int64_t)gridDim.x * 16) {
        const int64_t r = R % P.pad_rows, bk = R / P.pad_rows, kh = bk % A.kv_heads, b = bk / A.kv_heads;
        if (r >= P.row_count) {   // rows that are not there have no weight
            if (lane == 0) stats[R] = RowStat{INFINITY, 0.0f};
            continue;
        }
        int64_t t, h;
        split_row(P, kh, (uint32_t)r, &t, &h);
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
            top = both_max(top);
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
// NW waves of 32 rows share tiles of 32 * KB keys; while a tile is worked on the next one arrives in LDS.  With P.splits > 1 each split leaves
// its f32 part of dQ at part + split * (all of dQ).
template <typename T, int DP, int NW, int KB>
__global__ __launch_bounds__(64 * NW, 2) void attend_grad_q_kernel(artread_attend_t A, artread_attend_grads_t G,
                                                                    AttendPlan P, const RowStat* __restrict__ stats,
                                                                    float* __restrict__ part) {
    constexpr int TILE = 32 * KB * DP;
    __shared__ __attribute__((aligned(1024))) T ring[4][TILE];   // two tiles of K, two of V
    typedef typename Mma<T>::V8 V8;
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = uniform(threadIdx.x >> 6);
    const int dim = (int)A.dim;
    TileFetch<T, DP, KB, NW> fetcher;
    fetcher.start(wave);
    if (dim < DP) {
        for (int i = threadIdx.x; i < 4 * TILE / 8; i += 64 * NW) ((u32x4*)&ring[0][0])[i] = u32x4{0, 0, 0, 0};
        __syncthreads();
    }
    const int64_t total = P.items * P.splits;
    for (int64_t id = blockIdx.x; id < (total + 7) / 8 * 8; id += gridDim.x) {
        const int64_t w = xcd_item(id, total);
        if (w >= total) continue;
        if (id != blockIdx.x) {   // the tiles of the item before are read
            dma_wait<0>();
            wave_meet();
        }
        const int64_t rb = w % P.row_blocks, other = w / P.row_blocks;
        const int split = (int)(other % P.splits);
        const int64_t bk = other / P.splits, kh = bk % A.kv_heads, b = bk / A.kv_heads;
        const int64_t r = (rb * NW + wave) * 32 + (lane & 31);
        const T* kbase = (const T*)A.k + b * A.k_batch + kh * A.k_head;
        const T* vbase = (const T*)A.v + b * A.v_batch + kh * A.v_head;
        Walk<32 * KB> walk;   // of the tiles fetched; `left` of the one worked on
        walk.start(A, b, split, P.splits);
        auto fetch = [&](int stage) {   // keys of the tile, 0 behind the last
            if (!walk.settle()) return 0;
            const int left = walk.n - walk.j0;
            fetcher.fetch(kbase + walk.p * A.k_passage + walk.j0 * A.k_row, A.k_row, left, dim, lds_offset(ring[stage]));
            fetcher.fetch(vbase + walk.p * A.v_passage + walk.j0 * A.v_row, A.v_row, left, dim, lds_offset(ring[2 + stage]));
            walk.advance();
            return left;
        };
        int left = fetch(0);
        V8 q[DP / 16], g[DP / 16];
        load_q<T, DP>(A, P, (const T*)A.q, A.q_batch, A.q_row, A.q_head, b, kh, r, half, P.q_and, P.q_xor, q);
        load_q<T, DP>(A, P, (const T*)G.grad_out, G.g_batch, G.g_row, G.g_head, b, kh, r, half, 0xffffffffu, 0u, g);
        RowStat st{INFINITY, 0.0f};
        if (r < P.row_count) st = stats[bk * P.pad_rows + r];
        f32x16 acc[DP / 32];
        Spread<T> spread;
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) acc[db] = f32x16{};
        int stage = 0;
        while (left) {
            dma_wait<0>();
            wave_meet();   // everyone's pieces are there, and everyone is done with the tile before
            const int next = fetch(stage ^ 1);
            const uint32_t krow = opaque(lds_offset(ring[stage]) + rows_base<DP>(lane));
            const uint32_t kcol = opaque(lds_offset(ring[stage]) + columns_base<DP>(lane));
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
                for (int k = 0; k < DP / 16; ++k) {
                    s = Mma<T>::mul(lds_rows<T, DP>(krow, kb, k), q[k], s);
                    dp = Mma<T>::mul(lds_rows<T, DP>(krow, 2 * KB + kb, k), g[k], dp);
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], P.c, -st.x)) * (dp[i] - st.delta);
                if (left < 32 * KB) {
                    const int mine = left - 4 * half;
                    asm volatile("");   // a branch: most tiles are whole
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (32 * kb + 8 * (i >> 2) + (i & 3) >= mine) s[i] = 0.0f;
                }
                spread.fit(s, acc);
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
                    const V8 ds = weights8<T>(s, ks);
#pragma unroll
                    for (int db = 0; db < DP / 32; ++db)
                        acc[db] = Mma<T>::mul(lds_columns<T, DP>(kcol, 32 * kb + 16 * ks, db), ds, acc[db]);
                }
            }
            left = next;
            stage ^= 1;
        }
        if (r < P.row_count) {
            int64_t t, h;
            split_row(P, kh, (uint32_t)r, &t, &h);
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
// Four waves of 32 keys of one passage share tiles of 32 rows of Q and dO, fetched two tiles ahead into a ring of
// three in LDS: each is read as rows for S and dP and transposed for dK and dV.  With P.splits > 1 the rows are dealt
// to splits, which leave f32 parts of dK and dV.
template <typename T, int DP>
__global__ __launch_bounds__(256, 2) void attend_grad_kv_kernel(artread_attend_t A, artread_attend_grads_t G,
                                                                  AttendPlan P, const RowStat* __restrict__ stats,
                                                                  float* __restrict__ part) {
    constexpr int STAGES = 3;
    __shared__ __attribute__((aligned(1024))) T qtile[2 * STAGES][32 * DP];   // Q's tiles and behind them dO's
    __shared__ __attribute__((aligned(1024))) RowStat stile[STAGES][4][32];   // a copy for each wave
    typedef typename Mma<T>::V8 V8;
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = uniform(threadIdx.x >> 6);
    const int dim = (int)A.dim;
    const int64_t key_blocks = (A.len + 127) / 128;
    const int64_t total = P.items * P.splits;   // batch x passages x key_blocks x kv_heads x splits
    for (int64_t id = blockIdx.x; id < (total + 7) / 8 * 8; id += gridDim.x) {
        // Many rows: the workgroups of one key head stand together on an XCD, whose L2 then serves its rows.  Few:
        // the key heads of a state, neighbours in memory, are read side by side.
        int64_t item = P.by_head ? xcd_item(id, total) : id;
        if (item >= total) continue;
        if (id != blockIdx.x) {   // the tiles of the item before are read
            dma_wait<0>();
            wave_meet();
        }
        const int split = (int)(item % P.splits);
        item /= P.splits;
        int64_t kh = 0;
        if (!P.by_head) {
            kh = item % A.kv_heads;
            item /= A.kv_heads;
        }
        const int64_t j0 = item % key_blocks * 128;
        item /= key_blocks;
        const int64_t p = item % A.passages;
        item /= A.passages;
        if (P.by_head) {
            kh = item % A.kv_heads;
            item /= A.kv_heads;
        }
        const int64_t b = item;
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
            // pieces of 1 KiB: PR rows each, PW of a tile for each wave; rows that are not there repeat the last one
            // (their weight is zero), columns behind dim the first (they meet zeros of K and V)
            constexpr int CH = DP / 8, PR = 64 / CH, PW = 32 / PR / 4;
            const int prow = lane / CH, tiles = (int)((P.row_count + 31) / 32);
            const RowStat* sp = stats + (b * A.kv_heads + kh) * P.pad_rows;
            const T* qb = (const T*)A.q + b * A.q_batch + kh * P.share * A.q_head;
            const T* gb = (const T*)G.grad_out + b * G.g_batch + kh * P.share * G.g_head;
            auto fetch = [&](int tile, int stage) {
                int64_t t0, h0;
                split_row(P, 0, (uint32_t)tile * 32, &t0, &h0);
#pragma unroll
                for (int x = 0; x < PW; ++x) {
                    const int piece = wave * PW + x, row = piece * PR + prow;
                    int64_t r = (int64_t)tile * 32 + row, t, h;
                    r = r < P.row_count ? r : P.row_count - 1;
                    split_row(P, 0, (uint32_t)r, &t, &h);
                    int col = tile_chunk<DP>(row, lane % CH) * 8;
                    col = col < dim ? col : 0;
                    // bytes from the tile's first query position: a tile spans at most 32 of them
                    const uint32_t dt = (uint32_t)t - (uint32_t)t0;
                    dma16(qb + t0 * A.q_row, (dt * (uint32_t)A.q_row + (uint32_t)(h * A.q_head) + col) * 2, lds_offset(&qtile[stage][piece * 512]));
                    dma16(gb + t0 * G.g_row, (dt * (uint32_t)G.g_row + (uint32_t)(h * G.g_head) + col) * 2, lds_offset(&qtile[STAGES + stage][piece * 512]));
                }
                dma4(sp + tile * 32, (uint32_t)lane * 4, lds_offset(&stile[stage][wave][0]));
            };
            constexpr int LOADS = 2 * PW + 1;
            if (split < tiles) fetch(split, 0);
            if (split + P.splits < tiles) fetch(split + P.splits, 1);
            // one loop for waves with keys and one for those without: both load and meet at the barriers
            auto go = [&](auto with_keys) {
                int stage = 0;
                for (int tile = split; tile < tiles; tile += P.splits) {
                    if (tile + P.splits < tiles) dma_wait<LOADS>();   // all but the next tile's
                    else dma_wait<0>();
                    wave_meet();   // everyone's pieces are there, and everyone is done with the tile before
                    const int ahead = stage == 0 ? 2 : stage - 1;
                    if (tile + 2 * P.splits < tiles) fetch(tile + 2 * P.splits, ahead);
                    if constexpr (decltype(with_keys)::value) {
                        const uint32_t qrow = opaque(lds_offset(qtile[stage]) + rows_base<DP>(lane));
                        const uint32_t qcol = opaque(lds_offset(qtile[stage]) + columns_base<DP>(lane));
                        f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
                        for (int k = 0; k < DP / 16; ++k) {
                            s = Mma<T>::mul(lds_rows<T, DP>(qrow, 0, k), kf[k], s);
                            dp = Mma<T>::mul(lds_rows<T, DP>(qrow, STAGES, k), vf[k], dp);
                        }
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const float4 a = *(const float4*)&stile[stage][wave][8 * x + 4 * half];
                            const float4 c = *(const float4*)&stile[stage][wave][8 * x + 4 * half + 2];
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
                                dv[db] = Mma<T>::mul(lds_columns<T, DP>(qcol, STAGES * 32 + 16 * ks, db), pw, dv[db]);
                                dk[db] = Mma<T>::mul(lds_columns<T, DP>(qcol, 16 * ks, db), ds, dk[db]);
                            }
                        }
                    }
                    stage = stage == 2 ? 0 : stage + 1;
                }
            };
            if (j0 + 32 * wave < n) go(std::true_type{});   // uniform over the wave
            else go(std::false_type{});
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
