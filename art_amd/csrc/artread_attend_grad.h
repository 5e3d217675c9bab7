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

// 16 lanes per row, eight columns each.  The rows of a key head are padded to whole tiles of 64.  Bound by reading
// grad_out, out and rest: 8 x 1,024 rows of 16 x 128 bf16 in 19 us, 5.3 TB/s.
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

// The same with one power of two for a whole wave's dS, where its columns are not the accumulators' ones.  Beside the
// largest dS of the wave's walk so far, entries down to 2^-23 of it keep f16's bits in their two terms; what lies 2^-35
// below it is lost.
template <typename T>
struct SpreadAll {
    __device__ __forceinline__ float inverse() const { return 1.0f; }
    __device__ __forceinline__ float times(float x) const { return x; }
    template <int N>
    __device__ __forceinline__ void fit(const f32x16&, f32x16 (&)[N]) {}
};
template <>
struct SpreadAll<f16> {
    float f = 1.0f, most = 0.0f;
    __device__ __forceinline__ float inverse() const { return 1.0f / f; }
    __device__ __forceinline__ float times(float x) const { return x * f; }
    template <int N>
    __device__ __forceinline__ void fit(const f32x16& ds, f32x16 (&acc)[N]) {
        float top = fabsf(ds[0]);
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, fabsf(ds[i]));
        if (__any(top > most)) {
#pragma unroll
            for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
            int e = 10 - ilogbf(top);
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
};

// dS as two terms, the rounded value and what the rounding took, for products that share the other operand's LDS read.
// With one term the error of dQ is up to 1.5 times that of its own rounding, where a row's sum hangs on few keys; with
// two it is that rounding (48 rows, 100 x 250 states of 64 f16: 2.08e-4 instead of 3.1e-4).  It costs the row walk an
// eighth to a sixth of its time.  The key walk takes one: its sums run over more than 32 rows, 1.4 times, and the
// registers of a second term would spill (640 us instead of 510).  P takes one everywhere.
template <typename T>
__device__ __forceinline__ void terms8(const f32x16& s, int ks, typename Mma<T>::V8& hi, typename Mma<T>::V8& lo) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        hi[e] = (T)s[8 * ks + e];
        lo[e] = (T)(s[8 * ks + e] - (float)hi[e]);
    }
}

template <typename T>
__device__ __forceinline__ void put4(T* p, const float* x) {
    Vec<T, 4> w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w.x[e] = (T)x[e];
    store_vec<T, 4>(p, w);
}

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <typename T>
__device__ __forceinline__ u32x2 pack4(float a, float b, float c, float d) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    const T4 w = {(T)a, (T)b, (T)c, (T)d};
    return __builtin_bit_cast(u32x2, w);
}

// Accumulators of 32 keys (lane: key, elements: columns), times f, rounded, as rows: through 4 KiB of LDS of the
// wave's own, 64 columns at a time, so that eight lanes hold 128 bytes of a row.  Stores of 8 bytes by 64 rows would
// ask the L2 for eight times as many writes, which bound the gradient of few rows (456 us against 292 for 48 rows of 100 x 250 states).
// w[4 * c + x]: row 8 * x + (lane >> 3), columns 64 * c + 8 * (lane & 7)..
template <typename T, int DP>
__device__ __forceinline__ void turn_keys(const f32x16 (&acc)[DP / 32], float f, bool key, uint32_t lds, int lane,
                                          u32x4 (&w)[DP / 16]) {
    typedef __attribute__((address_space(3))) u32x2 lds_u32x2;
    const int ln = (int)opaque(lane), row = ln & 31;
#pragma unroll
    for (int c = 0; c < DP / 64; ++c) {
#pragma unroll
        for (int y = 0; y < 8; ++y) {
            const f32x16& v = acc[2 * c + (y >> 2)];
            const int i = 4 * (y & 3);
            u32x2 t = pack4<T>(f * v[i], f * v[i + 1], f * v[i + 2], f * v[i + 3]);
            if (!key) t = u32x2{0, 0};   // behind the length: zeros, whatever the accumulators hold
            *(lds_u32x2*)(uintptr_t)(lds + (uint32_t)(row * 128 + ((y ^ (row & 7)) * 16) + (ln >> 5) * 8)) = t;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int r = 8 * x + (ln >> 3);
            w[4 * c + x] = *(__attribute__((address_space(3))) u32x4*)(uintptr_t)(lds + (uint32_t)(r * 128 + (((ln & 7) ^ (r & 7)) * 16)));
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}
// and their way to memory: at(row) is the first element of row `row` of the 32, for those below `rows`
template <typename T, int DP>
__device__ __forceinline__ void store_turned(T* first, int64_t stride, int rows, int dim, int lane, const u32x4 (&w)[DP / 16]) {
    const int ln = (int)opaque(lane), d = 8 * (ln & 7);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        const int r = 8 * x + (ln >> 3);
#pragma unroll
        for (int c = 0; c < DP / 64; ++c)
            if (r < rows && 64 * c + d < dim) *(u32x4*)(first + r * stride + 64 * c + d) = w[4 * c + x];
    }
}

// The order of N products whose operands take R LDS reads each: the reads of A products ahead, of which the scheduler by
// itself keeps one.  Nothing else moves in or out: registers for more are not there.
template <int N, int R, int A>
__device__ __forceinline__ void ahead() {
    __builtin_amdgcn_sched_group_barrier(0x100, R * A, 0);
#pragma unroll
    for (int k = 0; k < N - A; ++k) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, A, 0);
    __builtin_amdgcn_sched_barrier(0);
}

// ---- dQ: the row walk -----------------------------------------------------------------------------------
// NW waves of 32 rows share tiles of 32 * KB keys; while a tile is worked on the next one arrives in LDS.  With
// P.splits > 1 each split leaves its f32 part of dQ at part + split * (all of dQ).  Bound by the matrix units and what
// stands between their products: 8 x 8 x 512 states of 128 bf16 columns, 75 % valid, 4,096 rows a key head in 440-460 us,
// 900-940 TFLOP/s with the second term's products; a product runs in 52 % of the cycles.  Four waves; for up to 64 rows one
// wave a workgroup, since the others would have none.
template <typename T, int DP, int NW, int KB>
__global__ __launch_bounds__(64 * NW, DP == 64 ? 3 : 2) void attend_grad_q_kernel(artread_attend_t A, artread_attend_grads_t G,
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
    const int64_t w = xcd_item(block_id(), total);
    if (w >= total) return;
    const int64_t rb = w % P.row_blocks, other = w / P.row_blocks;
    const int split = (int)(other % P.splits);
    const int64_t hb = other / P.splits, kh = hb / A.batch, b = hb % A.batch;
    const int64_t r = (rb * NW + wave) * 32 + (lane & 31);
    const T* kbase = (const T*)A.k + b * A.k_batch + kh * A.k_head + fetcher.first(A.k_row);
    const T* vbase = (const T*)A.v + b * A.v_batch + kh * A.v_head + fetcher.first(A.v_row);
    Walk<32 * KB> walk;   // of the tiles fetched
    walk.start(A, P, b, split, P.splits);
    uint64_t mask = 0, next_mask = 0;   // of the tile worked on, and of the one being fetched
    const T *kp = kbase, *vp = vbase;   // of the tile to fetch
    const int64_t kstep = walk.step * A.k_row, vstep = walk.step * A.v_row;
    auto fetch = [&](int stage) {
        if (!walk.settle()) return false;
        if (walk.moved) {
            kp = kbase + walk.p * A.k_passage + walk.j0 * A.k_row;
            vp = vbase + walk.p * A.v_passage + walk.j0 * A.v_row;
        }
        next_mask = walk.mask;
        fetcher.fetch(kp, A.k_row, next_mask, dim, lds_offset(ring[stage]));
        fetcher.fetch(vp, A.v_row, next_mask, dim, lds_offset(ring[2 + stage]));
        kp += kstep;
        vp += vstep;
        walk.advance();
        return true;
    };
    bool more = fetch(0);
    V8 q[DP / 16], g[DP / 16];
    load_q<T, DP>(A, P, (const T*)A.q, A.q_batch, A.q_row, A.q_head, b, kh, r, half, P.q_and, P.q_xor, q);
    load_q<T, DP>(A, P, (const T*)G.grad_out, G.g_batch, G.g_row, G.g_head, b, kh, r, half, 0xffffffffu, 0u, g);
    RowStat st{INFINITY, 0.0f};
    if (r < P.row_count) st = stats[(b * A.kv_heads + kh) * P.pad_rows + r];
    f32x16 acc[DP / 32];
    Spread<T> spread;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) acc[db] = f32x16{};
    int stage = 0;
    while (more) {
        mask = next_mask;
        dma_wait<0>();
        wave_meet();   // everyone's pieces are there, and everyone is done with the tile before
        more = fetch(stage ^ 1);
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
            if constexpr (DP == 128) {   // LDS reads eight products ahead: 1 to 3 % at 4,096 rows
                __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
#pragma unroll
                for (int k = 0; k < DP / 8 - 8; ++k) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                }
                __builtin_amdgcn_sched_group_barrier(0x008, 8, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], P.c, -st.x)) * (dp[i] - st.delta);
            if (!whole_tile<KB>(mask)) {
                const uint32_t mine = (uint32_t)(mask >> (32 * kb + 4 * half));
                asm volatile("");   // a branch: most tiles are whole
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (!(mine & (1u << (8 * (i >> 2) + (i & 3))))) s[i] = 0.0f;
            }
            spread.fit(s, acc);
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                V8 hi, lo;
                terms8<T>(s, ks, hi, lo);
#pragma unroll
                for (int db = 0; db < DP / 32; ++db) {
                    const V8 a = lds_columns<T, DP>(kcol, 32 * kb + 16 * ks, db);
                    acc[db] = Mma<T>::mul(a, hi, acc[db]);
                    acc[db] = Mma<T>::mul(a, lo, acc[db]);
                }
            }
        }
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

// ---- dK and dV: the key walk ------------------------------------------------------------------------------
// Four waves of 32 keys each share tiles of 64 rows of Q and dO; the next tile's loads to LDS are sent before a tile is
// worked on.  Each is read as rows for S and dP and transposed for dK and dV.  With P.splits > 1 the rows are dealt
// to splits, which leave f32 parts of dK and dV.  K, V, dK and dV of 32 keys are 192 registers of 256, so operands are few
// ahead: 455-490 us for 8 x 8 x 512 states of 128 bf16 columns, 75 % valid, 4,096 rows a key head, 840-910 TFLOP/s, a
// product in 48 % of the cycles.  The rest is waits, for LDS and for the next tile: the compiler, which does not count the
// loads to LDS, waits for the wave's own K and V at their first use in the loop (vmcnt(1) and vmcnt(0) for f16), behind
// the next tile's ten loads, so that a tile's first products wait for nearly all of the next one.
// Tile `first` + wave of a batch entry's tiles of 32 keys.  At 128 columns those with valid keys come first, so that the
// waves of a workgroup have keys whatever the lengths are: there two waves share a SIMD, and one without keys leaves half
// of it idle (128 rows, 100 x 150 states, 62 % valid: dQ, dK and dV 640 us instead of 797 with four tiles of one passage a
// workgroup).  At 64, where three do, finding such a tile costs as much as the idle waves (244 us instead of 239 for 128
// rows, 100 x 100 states): they are taken in the order they have in memory, as they are where a batch entry has more than
// kDealPassages of them, since every workgroup looks at their lengths.
constexpr int kDealPassages = 1024;
struct KeyTile {
    int p, j, n;   // passage (A.passages: none left), tile of it, its length
    bool some;     // a wave of the workgroup has valid keys
};
template <bool DEAL>
__device__ __forceinline__ KeyTile find_tile(const artread_attend_t& A, const AttendPlan& P, int64_t b, int per_passage,
                                             int first, int wave) {
    const int slot = first + wave, passages = (int)A.passages, len = (int)A.len;
    const int32_t* lengths = A.lengths && !P.pack ? A.lengths + b * A.passages : nullptr;
    const int lane = threadIdx.x & 63;
    if (!DEAL || !lengths || passages > kDealPassages) {   // the lanes look at one tile each
        const int p = (first + (lane & 3)) / per_passage, j = first + (lane & 3) - p * per_passage;
        int n = p < passages ? len : 0;
        if (lengths && p < passages) n = lengths[p];
        n = n < 0 ? 0 : (n < len ? n : len);
        const bool some = __any(32 * j < n);
        return KeyTile{__builtin_amdgcn_readlane(p, wave), __builtin_amdgcn_readlane(j, wave), __builtin_amdgcn_readlane(n, wave), some};
    }
    int valid = 0, before = 0;
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {   // tiles with valid keys, then those without
        before = pass ? valid : 0;
        for (int p0 = 0; p0 < passages; p0 += 64) {
            const int p = p0 + lane;
            int n = p < passages ? lengths[p] : 0;
            n = n < 0 ? 0 : (n < len ? n : len);
            int c = (n + 31) >> 5;
            if (pass) c = p < passages ? per_passage - c : 0;
            int sum = c;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int x = __shfl_up(sum, o);
                if (lane >= o) sum += x;
            }
            const uint64_t behind = __ballot(before + sum > slot);
            if (behind) {
                const int l = __ffsll((unsigned long long)behind) - 1;
                const int j = slot - (before + __builtin_amdgcn_readlane(sum - c, l));
                const int m = __builtin_amdgcn_readlane(n, l);
                return KeyTile{p0 + l, pass ? j + (per_passage - __builtin_amdgcn_readlane(c, l)) : j, m, !pass || first < valid};
            }
            before += __builtin_amdgcn_readlane(sum, 63);
        }
        if (!pass) valid = before;
    }
    return KeyTile{passages, 0, 0, first < valid};
}

template <typename T, int DP>
__global__ __launch_bounds__(256, 2) void attend_grad_kv_kernel(artread_attend_t A, artread_attend_grads_t G,
                                                                  AttendPlan P, const RowStat* __restrict__ stats,
                                                                  float* __restrict__ part) {
    constexpr int RT = 2, TILE = 32 * RT * DP;
    __shared__ __attribute__((aligned(1024))) T qtile[4][TILE];               // two tiles of Q, two of dO
    __shared__ __attribute__((aligned(1024))) RowStat stile[2][4][32 * RT];   // a copy for each wave
    typedef typename Mma<T>::V8 V8;
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = uniform(threadIdx.x >> 6);
    const int dim = (int)A.dim;
    const int per_passage = (int)((A.len + 31) / 32);
    const int64_t groups = (A.passages * per_passage + 3) / 4;
    const int64_t total = P.items * P.splits;   // batch x kv_heads x groups x splits
    const int64_t id = block_id();
    // Many rows: the workgroups of one key head stand together on an XCD, whose L2 then serves its rows.  Few:
    // the key heads of a state, neighbours in memory, are read side by side.
    int64_t item = P.by_head ? xcd_item(id, total) : id;
    if (item >= total) return;
    const int split = (int)(item % P.splits);
    item /= P.splits;
    int64_t kh = 0;
    if (!P.by_head) {
        kh = item % A.kv_heads;
        item /= A.kv_heads;
    }
    const int first = (int)(item % groups) * 4;
    item /= groups;
    if (P.by_head) {
        kh = item % A.kv_heads;
        item /= A.kv_heads;
    }
    const int64_t b = item;
    const KeyTile at_tile = find_tile<DP == 128>(A, P, b, per_passage, first, wave);
    const int64_t p = at_tile.p, j1 = 32 * at_tile.j, j = j1 + (lane & 31);   // this lane's key
    bool key = j < at_tile.n;   // never where no tile is left
    if (P.pack && key) {
        Packed packed;
        packed.start(A, P, b);
        packed.ask((int)j);
        key = packed.valid();
    }
    f32x16 dk[DP / 32], dv[DP / 32];
    Spread<T> spread;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) dk[db] = dv[db] = f32x16{};
    if (at_tile.some) {   // uniform over the workgroup
        if (dim < DP) {
            for (int i = threadIdx.x; i < 4 * TILE / 8; i += 256) ((u32x4*)&qtile[0][0])[i] = u32x4{0, 0, 0, 0};
            __syncthreads();
        }
        V8 kf[DP / 16], vf[DP / 16];
        const T* kp = (const T*)A.k + b * A.k_batch + p * A.k_passage + j * A.k_row + kh * A.k_head + 8 * half;
        const T* vp = (const T*)A.v + b * A.v_batch + p * A.v_passage + j * A.v_row + kh * A.v_head + 8 * half;
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            const bool ok = key && 16 * s + 8 * half < dim;
            kf[s] = load8<T>(kp + 16 * s, ok);
            vf[s] = load8<T>(vp + 16 * s, ok);
        }
        // pieces of 1 KiB, PR rows each, every fourth of a tile by one wave: 4 * PR rows from one to the next.  Where that
        // is whole query positions, a lane's pieces of all whole tiles lie at one offset from uniform addresses.
        constexpr int CH = DP / 8, PR = 64 / CH, PW = 32 * RT / PR / 4;
        const int tiles = (int)((P.row_count + 32 * RT - 1) / (32 * RT));
        const RowStat* sp = stats + (b * A.kv_heads + kh) * P.pad_rows;
        const T* qb = (const T*)A.q + b * A.q_batch + kh * P.share * A.q_head;
        const T* gb = (const T*)G.grad_out + b * G.g_batch + kh * P.share * G.g_head;
        const uint32_t positions = 4 * PR / P.share;
        const bool even = positions * P.share == 4 * PR && dim == DP;
        auto fetch = [&](int tile, int stage) {
            int64_t t0, h0, t, h;
            split_row(P, 0, (uint32_t)tile * 32 * RT, &t0, &h0);
            const uint32_t ln = opaque(lane), prow = ln / CH;
            const uint32_t dst = lds_offset(&qtile[stage][wave * 512]), chunk = tile_chunk<DP>(prow, ln % CH) ^ (DP == 128 ? wave : (wave & 1) << 1);
            const T *qt = qb + t0 * A.q_row, *gt = gb + t0 * G.g_row;
            if (even && (int64_t)(tile + 1) * 32 * RT <= P.row_count) {   // uniform
                split_row(P, 0, wave * PR + prow, &t, &h);
                uint32_t qo[PW], go[PW];
#pragma unroll
                for (int x = 0; x < PW; ++x) {
                    qo[x] = ((uint32_t)t * (uint32_t)A.q_row + (uint32_t)(h * A.q_head) + chunk * 8) * 2;
                    go[x] = ((uint32_t)t * (uint32_t)G.g_row + (uint32_t)(h * G.g_head) + chunk * 8) * 2;
                }
                dma_pieces<PW, 4096>(qt, positions * (uint32_t)A.q_row * 2, qo, dst);
                dma_pieces<PW, 4096>(gt, positions * (uint32_t)G.g_row * 2, go, dst + 2 * TILE * 2);
            } else {
                const bool there = dim == DP || chunk * 8 < (uint32_t)dim;   // columns behind dim stay cleared
#pragma unroll
                for (int x = 0; x < PW; ++x) {
                    const int64_t r = (int64_t)tile * 32 * RT + (x * 4 + wave) * PR + prow;
                    split_row(P, 0, (uint32_t)r, &t, &h);
                    // bytes from the tile's first query position: a tile spans at most as many of them as rows
                    const uint32_t dt = (uint32_t)t - (uint32_t)t0;
                    if (there && r < P.row_count) {
                        dma16(qt, (dt * (uint32_t)A.q_row + (uint32_t)(h * A.q_head) + chunk * 8) * 2, dst + x * 4096);
                        dma16(gt, (dt * (uint32_t)G.g_row + (uint32_t)(h * G.g_head) + chunk * 8) * 2, dst + 2 * TILE * 2 + x * 4096);
                    }
                }
                if ((int64_t)(tile + 1) * 32 * RT > P.row_count) {   // uniform
                    // rows that are not there: the last one's query, whose weight is zero, and a gradient of zeros, since no
                    // weight times an infinite one would be NaN
                    const uint32_t l2 = opaque(lane), z = opaque(0);   // made here: no register holds them over the loop
                    const int left = (int)(P.row_count - (int64_t)tile * 32 * RT) - (int)(wave * PR + l2 / CH);
                    split_row(P, 0, (uint32_t)(P.row_count - 1), &t, &h);
                    const uint32_t last = (((uint32_t)t - (uint32_t)t0) * (uint32_t)A.q_row + (uint32_t)(h * A.q_head) + chunk * 8) * 2;
#pragma unroll
                    for (int x = 0; x < PW; ++x)
                        if (x * 4 * PR >= left) {
                            if (there) dma16(qt, last, dst + x * 4096);
                            *(__attribute__((address_space(3))) u32x4*)(uintptr_t)(dst + 2 * TILE * 2 + x * 4096 + l2 * 16) = u32x4{z, z, z, z};
                        }
                }
            }
#pragma unroll
            for (int x = 0; x < RT; ++x)   // the statistics are padded to whole tiles
                dma4(sp + tile * 32 * RT + 32 * x, ln * 4, lds_offset(&stile[stage][wave][32 * x]));
        };
        if (split < tiles) fetch(split, 0);
        // one loop for waves with keys and one for those without: both load and meet at the barriers
        auto go = [&](auto with_keys) {
            int stage = 0;
            for (int tile = split; tile < tiles; tile += P.splits) {
                dma_wait<0>();
                wave_meet();   // everyone's pieces are there, and everyone is done with the tile before
                if (tile + P.splits < tiles) fetch(tile + P.splits, stage ^ 1);
                if constexpr (decltype(with_keys)::value) {
                    const uint32_t qrow = opaque(lds_offset(qtile[stage]) + rows_base<DP>(lane));
                    const uint32_t qcol = opaque(lds_offset(qtile[stage]) + columns_base<DP>(lane));
#pragma unroll
                    for (int x = 0; x < RT; ++x) {
                        f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
                        for (int k = 0; k < DP / 16; ++k) {
                            s = Mma<T>::mul(lds_rows<T, DP>(qrow, x, k), kf[k], s);
                            dp = Mma<T>::mul(lds_rows<T, DP>(qrow, 2 * RT + x, k), vf[k], dp);
                        }
                        ahead<DP / 8, 1, DP == 128 ? 2 : 4>();
#pragma unroll
                        for (int y = 0; y < 4; ++y) {
                            const float4 a = *(const float4*)&stile[stage][wave][32 * x + 8 * y + 4 * half];
                            const float4 c = *(const float4*)&stile[stage][wave][32 * x + 8 * y + 4 * half + 2];
                            const float xs[4] = {a.x, a.z, c.x, c.z}, ds[4] = {a.y, a.w, c.y, c.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int i = 4 * y + e;
                                s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], P.c, -xs[e]));
                                dp[i] = s[i] * (dp[i] - ds[e]);
                            }
                        }
                        spread.fit(dp, dk);
                        V8 pw[2], ds[2];
#pragma unroll
                        for (int ks = 0; ks < 2; ++ks) {
                            pw[ks] = weights8<T>(s, ks);
                            ds[ks] = weights8<T>(dp, ks);
                        }
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                            for (int db = 0; db < DP / 32; ++db) {
                                dv[db] = Mma<T>::mul(lds_columns<T, DP>(qcol, 32 * (2 * RT + x) + 16 * ks, db), pw[ks], dv[db]);
                                dk[db] = Mma<T>::mul(lds_columns<T, DP>(qcol, 32 * x + 16 * ks, db), ds[ks], dk[db]);
                            }
                        ahead<DP / 8, 2, 4>();
                    }
                }
                stage ^= 1;
            }
        };
        if (__any(key)) go(std::true_type{});   // uniform over the wave
        else go(std::false_type{});
    }
    const int64_t all = A.batch * A.passages * A.len * A.kv_heads * dim;
    const float fv = P.unweight, fk = A.scale * spread.inverse() * P.unweight;
    if (P.splits == 1) {
        __syncthreads();   // the tiles are read
        const uint32_t own = lds_offset(&qtile[0][0]) + (uint32_t)wave * 4096;
        const int64_t at = (((b * A.passages + p) * A.len + j1) * A.kv_heads + kh) * dim;
        const int rows = p >= A.passages ? 0 : (A.len - j1 < 32 ? (int)(A.len - j1) : 32);
        u32x4 w[DP / 16];
        turn_keys<T, DP>(dv, fv, key, own, lane, w);
        store_turned<T, DP>((T*)G.grad_v + at, A.kv_heads * dim, rows, dim, lane, w);
        turn_keys<T, DP>(dk, fk, key, own, lane, w);
        store_turned<T, DP>((T*)G.grad_k + at, A.kv_heads * dim, rows, dim, lane, w);
        return;
    }
    if (p >= A.passages || j >= A.len) return;
    const int64_t at = (((b * A.passages + p) * A.len + j) * A.kv_heads + kh) * dim;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int d = 32 * db + 8 * x + 4 * half;
            if (d >= dim) continue;
            float yk[4], yv[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {   // behind the length: zeros, whatever the accumulators hold
                yk[e] = key ? fk * dk[db][4 * x + e] : 0.0f;
                yv[e] = key ? fv * dv[db][4 * x + e] : 0.0f;
            }
            *(float4*)(part + split * 2 * all + at + d) = make_float4(yk[0], yk[1], yk[2], yk[3]);
            *(float4*)(part + (split * 2 + 1) * all + at + d) = make_float4(yv[0], yv[1], yv[2], yv[3]);
        }
}

// ---- all three gradients at once: few rows -----------------------------------------------------------------
// Up to 32 * RB rows per key head.  A wave walks tiles of 32 keys, those behind the lengths among them (they get their
// zeros here), and finishes dK and dV of a tile before the next: every state is read once and every gradient written
// once, which is what bounds this, where the two walks would read the states twice (16 rows of 8 x 12 heads, 100 x 250
// states of 64 bf16, 75 % valid: 246 us, 4.4 TB/s; of 128 columns 470 us, 4.6 TB/s; 48 rows of 64 f16, 62 % valid: 275 to
// 310 us, 3.3 to 3.7 TB/s).  Two tiles of K in LDS, the next one on its way from the start of a tile, cost more workgroups
// than they save waiting (325 us against 294, fewer rows 2 % more).  S^T
// and dP^T leave P^T and dS^T as B operands over the keys, for dQ; dV and dK want them over the rows, so both go through a
// 32 x 32 tile of LDS and come back by the transposing read.  A tile's results are stored once the next tile has arrived,
// so that waiting for that tile does not wait for the stores; the compiler's own waits still do, at the first use of the
// row statistics and where a passage's length is read, and for 48 rows a wave waits in 46 % of its cycles.  Two row blocks
// in f16, and in bf16 where packed, fill the 256 registers: 4 to 10 of them are kept in scratch, and their loads, the zeros
// of a partly valid tile among them, wait for the stores and the pieces before them too.  The waves of a workgroup add
// their dQ in LDS, in order.  PACK: passages too short to fill tiles of their own are packed; a kernel of its own, for the
// registers.  At 64 columns two waves share a SIMD; at 128 LDS leaves one, with up to 436 registers.
template <typename T, int DP, int RB, int NW, bool PACK>
__global__ __launch_bounds__(64 * NW, DP == 64 ? 2 : 1) void attend_grad_stream_kernel(artread_attend_t A, artread_attend_grads_t G,
                                                                        AttendPlan P, const RowStat* __restrict__ stats,
                                                                        float* __restrict__ part) {
    constexpr int TILE = 32 * DP, CH = DP / 8;
    constexpr int SHARED = 2 * RB * TILE, OWN = 2 * TILE + 3 * 1024;   // elements: Q and dO; K, V, P and both terms of dS of a wave
    constexpr int BYTES = (SHARED + NW * OWN) * 2, SUMS = NW * 32 * RB * DP * 4;
    __shared__ __attribute__((aligned(1024))) char lds[BYTES > SUMS ? BYTES : SUMS];
    typedef typename Mma<T>::V8 V8;
    typedef __attribute__((address_space(3))) u32x2 lds_u32x2;
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = uniform(threadIdx.x >> 6);
    const int dim = (int)A.dim, len = (int)A.len;
    T* qtile = (T*)lds;
    T* gtile = qtile + RB * TILE;
    const uint32_t mine = lds_offset(lds) + (uint32_t)(SHARED + wave * OWN) * 2, pd = mine + 2 * TILE * 2;
    TileFetch<T, DP, 1, 1> fetcher;
    fetcher.start(0);
    const int per_passage = (len + 31) / 32;
    const int64_t total = P.items * P.splits;   // splits: workgroups per item
    const int64_t id = block_id();
    if (id >= total) return;
    const int group = (int)(id % P.splits);
    const int64_t bk = id / P.splits, kh = bk % A.kv_heads, b = bk / A.kv_heads;
    for (int i = threadIdx.x; i < RB * 32 * CH; i += 64 * NW) {
        const int row = i / CH, chunk = i % CH;
        // rows that are not there have no weight and no gradient; their scores repeat the last row's, since those of zeros
        // would be NaN for an infinite key that every row does without
        const bool there = row < P.row_count;
        int64_t t, h;
        split_row(P, kh, there ? (uint32_t)row : (uint32_t)(P.row_count - 1), &t, &h);
        const int at = row * DP + tile_chunk<DP>(row, chunk) * 8;
        *(V8*)(qtile + at) = load8<T>((const T*)A.q + b * A.q_batch + t * A.q_row + h * A.q_head + 8 * chunk, 8 * chunk < dim);
        *(V8*)(gtile + at) = load8<T>((const T*)G.grad_out + b * G.g_batch + t * G.g_row + h * G.g_head + 8 * chunk, there && 8 * chunk < dim);
    }
    if (dim < DP) {   // the columns behind dim of the wave's own tiles
        for (int i = lane; i < 2 * TILE / 8; i += 64)
            *(__attribute__((address_space(3))) u32x4*)(uintptr_t)(mine + i * 16) = u32x4{0, 0, 0, 0};
        // loads from memory to LDS do not wait for the wave's LDS stores: the first tile's come to the same places
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    RowStat st[RB];
    f32x16 dq[RB][DP / 32];
    Spread<T> spread_q[RB];
    SpreadAll<T> spread_k;
#pragma unroll
    for (int x = 0; x < RB; ++x) {
        st[x] = RowStat{INFINITY, 0.0f};
        if (32 * x < P.pad_rows) st[x] = stats[bk * P.pad_rows + 32 * x + (lane & 31)];
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) dq[x][db] = f32x16{};
    }
    const T* kbase = (const T*)A.k + b * A.k_batch + kh * A.k_head;
    const T* vbase = (const T*)A.v + b * A.v_batch + kh * A.v_head;
    const int step = P.splits * NW, step_p = step / per_passage, step_j = step % per_passage;
    int p = (group * NW + wave) / per_passage, jt = (group * NW + wave) % per_passage;
    uint32_t mask = 0;   // valid keys of the tile at p, jt; 0: nothing was fetched
    int chunk = -1, lengths = len;   // of 64 passages, one per lane
    Packed packed;
    if constexpr (PACK) {
        packed.start(A, P, b);
        packed.ask(32 * jt + (lane & 31));
    }
    auto fetch = [&]() {
        mask = 0;
        if (p >= (int)A.passages) return;
        if constexpr (PACK) {
            mask = (uint32_t)__ballot(packed.valid());
        } else {
            if (A.lengths && (p >> 6) != chunk) {   // rarely: a load here waits for the stores before it
                chunk = p >> 6;
                const int i = chunk * 64 + lane;
                lengths = i < (int)A.passages ? A.lengths[b * A.passages + i] : 0;
            }
            const int left = min(len, __builtin_amdgcn_readlane(lengths, p & 63)) - 32 * jt;
            mask = left <= 0 ? 0u : (left >= 32 ? ~0u : (1u << left) - 1);
        }
        if (!mask) return;
        fetcher.fetch(kbase + p * A.k_passage + (int64_t)32 * jt * A.k_row, A.k_row, mask, dim, mine);
        fetcher.fetch(vbase + p * A.v_passage + (int64_t)32 * jt * A.v_row, A.v_row, mask, dim, mine + TILE * 2);
    };
    f32x16 dk[DP / 32], dv[DP / 32];
    u32x4 wk[DP / 16], wv[DP / 16];   // the tile before's, rounded, and where it was
    int held_p = -1, held_j = 0;
    auto store = [&]() {
        if (held_p < 0) return;
        const int64_t at = (((b * A.passages + held_p) * A.len + held_j) * A.kv_heads + kh) * dim;
        store_turned<T, DP>((T*)G.grad_k + at, A.kv_heads * dim, len - held_j, dim, lane, wk);
        store_turned<T, DP>((T*)G.grad_v + at, A.kv_heads * dim, len - held_j, dim, lane, wv);
    };
    // dV and dK += the products of row block x, whose P and dS stand in LDS
    auto add_block = [&](int x) {
        const int i = lane & 15;
        const uint32_t pr = opaque(pd + (uint32_t)((4 * half + (i >> 2)) * 64 + (((((lane & 16) >> 2) + (i & 3)) ^ half) * 8)));
        const uint32_t qcol = opaque(lds_offset(qtile) + columns_base<DP>(lane));
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // they are written: LDS keeps a wave's order
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            V8 pk[3];
#pragma unroll
            for (int a = 0; a < 3; ++a) {
                union {
                    s16x4 h[2];
                    V8 v;
                } u;
#pragma unroll
                for (int y = 0; y < 2; ++y)
                    u.h[y] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(uintptr_t)(
                        (pr ^ (uint32_t)(32 * ks + 16 * y)) + (uint32_t)(a * 2048 + (16 * ks + 8 * y) * 64)));
                pk[a] = u.v;
            }
#pragma unroll
            for (int db = 0; db < DP / 32; ++db) {
                dv[db] = Mma<T>::mul(lds_columns<T, DP>(qcol, 32 * (RB + x) + 16 * ks, db), pk[0], dv[db]);
                const V8 a = lds_columns<T, DP>(qcol, 32 * x + 16 * ks, db);
                dk[db] = Mma<T>::mul(a, pk[1], dk[db]);
                dk[db] = Mma<T>::mul(a, pk[2], dk[db]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // and read
    };
    fetch();
    if constexpr (PACK) packed.ask(32 * (jt + step_j) + (lane & 31));
    __syncthreads();   // Q and dO are there
    while (true) {
        if (mask) dma_wait<0>();
        store();
        if (p >= (int)A.passages) break;
        held_p = p;
        held_j = 32 * jt;
        const uint32_t now = mask;
        if (now) {
            const uint32_t krow = opaque(mine + rows_base<DP>(lane));
            const uint32_t qrow = opaque(lds_offset(qtile) + rows_base<DP>(lane));
#pragma unroll
            for (int db = 0; db < DP / 32; ++db) dk[db] = dv[db] = f32x16{};
#pragma unroll
            for (int x = 0; x < RB; ++x) {
                if (x > 0) {   // dV and dK of the row block before
                    add_block(x - 1);
                    __builtin_amdgcn_sched_barrier(0);
                }
                f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
                for (int k = 0; k < DP / 16; ++k) {
                    s = Mma<T>::mul(lds_rows<T, DP>(krow, 0, k), lds_rows<T, DP>(qrow, x, k), s);
                    dp = Mma<T>::mul(lds_rows<T, DP>(krow, 1, k), lds_rows<T, DP>(qrow, RB + x, k), dp);
                }
                // operands two steps ahead and no further: more of them would not fit beside the accumulators
                __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
#pragma unroll
                for (int k = 0; k < DP / 16 - 2; ++k) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
                }
                __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], P.c, -st[x].x));
                    dp[i] = s[i] * (dp[i] - st[x].delta);
                }
                if (now != ~0u) {
                    const uint32_t keys = opaque(now >> (4 * half));
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (!(keys & (1u << (8 * (i >> 2) + (i & 3))))) dp[i] = 0.0f;
                }
                // P and dS to LDS as [row][key], 8-byte pieces permuted by the row
                const uint32_t pw = opaque(pd + (uint32_t)((lane & 31) * 64 + ((half ^ ((lane >> 2) & 7)) * 8)));
                spread_k.fit(dp, dk);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    *(lds_u32x2*)(uintptr_t)(pw ^ (16 * i)) = pack4<T>(s[4 * i], s[4 * i + 1], s[4 * i + 2], s[4 * i + 3]);
                    float y[4], z[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        y[e] = spread_k.times(dp[4 * i + e]);
                        z[e] = y[e] - (float)(T)y[e];
                    }
                    *(lds_u32x2*)(uintptr_t)((pw ^ (16 * i)) + 2048) = pack4<T>(y[0], y[1], y[2], y[3]);
                    *(lds_u32x2*)(uintptr_t)((pw ^ (16 * i)) + 4096) = pack4<T>(z[0], z[1], z[2], z[3]);
                }
                spread_q[x].fit(dp, dq[x]);
                const uint32_t kcol = opaque(mine + columns_base<DP>(lane));
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
                    V8 hi, lo;
                    terms8<T>(dp, ks, hi, lo);
#pragma unroll
                    for (int db = 0; db < DP / 32; ++db) {
                        const V8 a = lds_columns<T, DP>(kcol, 16 * ks, db);
                        dq[x][db] = Mma<T>::mul(a, hi, dq[x][db]);
                        dq[x][db] = Mma<T>::mul(a, lo, dq[x][db]);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // K and V are read: the next tile may come
        }
        p += step_p;
        jt += step_j;
        if (jt >= per_passage) {
            jt -= per_passage;
            ++p;
        }
        fetch();
        if constexpr (PACK) packed.ask(32 * (jt + step_j) + (lane & 31));   // one passage: the tile after, or none
        if (now) add_block(RB - 1);
        const float fk = A.scale * spread_k.inverse() * P.unweight;
        const bool key = now >> (lane & 31) & 1;
        turn_keys<T, DP>(dv, P.unweight, key, pd, lane, wv);
        turn_keys<T, DP>(dk, fk, key, pd, lane, wk);
    }
    // dQ of the workgroup: [wave][d][row]
    float* sums = (float*)lds;
    __syncthreads();
#pragma unroll
    for (int x = 0; x < RB; ++x) {
        const float f = A.scale * spread_q[x].inverse() * P.unweight;
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                sums[((wave * RB + x) * DP + 32 * db + 8 * (i >> 2) + 4 * half + (i & 3)) * 32 + (lane & 31)] = f * dq[x][db][i];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < RB * 32 * (DP / 4); i += 64 * NW) {
        const int row = i & 31, d = (i >> 5) % (DP / 4) * 4, x = i / (32 * (DP / 4)), r = 32 * x + row;
        if (r >= P.row_count || d >= dim) continue;
        float y[4] = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < NW; ++w)
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] += sums[((w * RB + x) * DP + d + e) * 32 + row];
        int64_t t, h;
        split_row(P, kh, (uint32_t)r, &t, &h);
        const int64_t at = ((b * A.rows + t) * A.heads + h) * dim + d;
        if (P.splits > 1) *(float4*)(part + group * (A.batch * A.rows * A.heads * dim) + at) = make_float4(y[0], y[1], y[2], y[3]);
        else put4<T>((T*)G.grad_q + at, y);
    }
}

// out = sum of `splits` f32 parts `stride` apart, in order, rounded once; n is a multiple of 8.  Five parts of 8 x 48 x 12
// rows of 64: 5 us, mostly a launch.
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
