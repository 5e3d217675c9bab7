// Embedding lookup of padded token rows and its gradient by sorted tokens (include/artread.h).
// Included by artread.hip only.
#pragma once
#include "artread_common.h"

// ---- what a position holds ------------------------------------------------------------------------
// Positions are numbered row * len + entry.  A position is valid iff its entry lies below its row's
// length and its token inside the vocabulary; its key is then the table row.
struct Tokens {
    const void* tokens;
    const int32_t* lengths;   // nullptr: all of len
    uint32_t len;
    uint32_t inv_len;         // floor(2^32 / len), 2^32 - 1 for len 1
    int64_t vocab;
    int64_t vocab_base;
    int64_t positions;        // n * len, below 2^31
};

// row and entry of a position: the quotient from inv_len is at most one too small, which the comparison mends
__device__ __forceinline__ void split_position(const Tokens& T, uint32_t pos, uint32_t* row, uint32_t* entry) {
    uint32_t q = __umulhi(pos, T.inv_len);
    uint32_t r = pos - q * T.len;
    if (r >= T.len) {
        q += 1;
        r -= T.len;
    }
    *row = q;
    *entry = r;
}

// the key of a position, -1 if it is not valid
template <typename IDX>
__device__ __forceinline__ int32_t key_of(const Tokens& T, uint32_t pos) {
    uint32_t row, entry;
    split_position(T, pos, &row, &entry);
    if (T.lengths && (int64_t)entry >= (int64_t)T.lengths[row]) return -1;
    const int64_t tok = (int64_t)((const IDX*)T.tokens)[pos];
    // the difference of two int64 with tok >= vocab_base always fits a uint64
    const uint64_t d = (uint64_t)tok - (uint64_t)T.vocab_base;
    return tok >= T.vocab_base && d < (uint64_t)T.vocab ? (int32_t)d : -1;
}

// ---- lookup ---------------------------------------------------------------------------------------
// A thread owns one chunk of EPV output elements (16 bytes where the layout allows, else one element)
// of U rows at a time; `cpr` chunks make a row, a workgroup holds `rpp` rows side by side.  The keys of
// its rows are requested before any table row, those before any store: three dependent round trips per
// U * rpp rows.  The table is read through the caches (a few thousand rows serve a whole batch), the
// output, which another kernel reads much later, is stored past them.
template <typename TT, typename OT, typename IDX, int EPV>
__global__ __launch_bounds__(256) void embed_kernel(const TT* __restrict__ table, int64_t table_stride, Tokens T,
                                                    float scale, OT* __restrict__ out, int dim, int cpr, int rpp) {
    constexpr int U = 8;
    const int r = cpr < 256 ? (int)threadIdx.x / cpr : 0;
    const int c0 = cpr < 256 ? (int)threadIdx.x - r * cpr : (int)threadIdx.x;
    if (r >= rpp) return;
    const int64_t step = (int64_t)gridDim.x * rpp * U;
    for (int64_t base = (int64_t)blockIdx.x * rpp * U + r; base < T.positions; base += step) {
        int32_t key[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t pos = base + (int64_t)u * rpp;
            key[u] = pos < T.positions ? key_of<IDX>(T, (uint32_t)pos) : -1;
        }
        for (int c = c0; c < cpr; c += 256) {
            Vec<TT, EPV> v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int e = 0; e < EPV; ++e) v[u].x[e] = from_f32<TT>(0.0f);
                if (key[u] >= 0) v[u] = load_vec<TT, EPV>(table + key[u] * table_stride + (int64_t)c * EPV);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t pos = base + (int64_t)u * rpp;
                if (pos >= T.positions) break;
                Vec<OT, EPV> w;
#pragma unroll
                for (int e = 0; e < EPV; ++e) w.x[e] = from_f32<OT>(key[u] >= 0 ? scale * to_f32(v[u].x[e]) : 0.0f);
                store_vec_nt<OT, EPV>(out + pos * dim + (int64_t)c * EPV, w);
            }
        }
    }
}

// ---- gradient: the sort ---------------------------------------------------------------------------
// A stable radix sort of the valid positions by key, least significant digit first, digits of at most
// nine bits (two passes for every vocabulary up to 262,144).  Stability makes the order of a token's
// positions, and with it every sum, a function of the tokens alone.  Per pass: digit counts of every
// block's chunk, then each block derives its own bases from all counts and places its chunk.
struct SortPlan {
    int blocks;       // chunks of the position list
    int64_t chunk;    // positions per chunk, a multiple of 256
    int bits;         // of a digit
    int passes;
};
struct SortMeta {
    uint32_t valid;   // valid positions
};
struct Pair {
    uint32_t key, pos;
};

template <typename IDX, bool FIRST>
__device__ __forceinline__ bool sort_item(const Tokens& T, const Pair* in, int64_t i, int64_t count, Pair* p) {
    if (i >= count) return false;
    if (FIRST) {
        const int32_t k = key_of<IDX>(T, (uint32_t)i);
        *p = Pair{(uint32_t)k, (uint32_t)i};
        return k >= 0;
    }
    *p = in[i];
    return true;
}

// digit counts [blocks][1 << bits]; the first pass also clears the marks of used table rows
template <typename IDX, bool FIRST>
__global__ __launch_bounds__(256) void sort_count_kernel(Tokens T, const Pair* __restrict__ in,
                                                         const SortMeta* __restrict__ meta, SortPlan P, int shift,
                                                         uint32_t* __restrict__ counts, uint8_t* __restrict__ used) {
    __shared__ uint32_t hist[512];
    const int digits = 1 << P.bits;
    for (int d = threadIdx.x; d < digits; d += 256) hist[d] = 0;
    __syncthreads();
    if (FIRST)
        for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (T.vocab + 15) / 16; i += (int64_t)gridDim.x * 256)
            ((uint4*)used)[i] = make_uint4(0, 0, 0, 0);   // the array is padded to 16 bytes
    const int64_t count = FIRST ? T.positions : (int64_t)meta->valid;
    const int64_t lo = blockIdx.x * P.chunk, hi = lo + P.chunk < count ? lo + P.chunk : count;
    for (int64_t i = lo + threadIdx.x; i < hi; i += 256) {
        Pair p;
        if (sort_item<IDX, FIRST>(T, in, i, hi, &p)) atomicAdd(&hist[(p.key >> shift) & (digits - 1)], 1u);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += 256) counts[(int64_t)blockIdx.x * digits + d] = hist[d];
}

// Places one chunk.  Each of the four waves owns a quarter of it and walks the quarter in order, 64
// positions at a time: the lanes that share a digit find each other by `bits` ballots, the lane's rank is
// the number of them below it, and the highest one moves the wave's next free place of that digit on.
template <typename IDX, bool FIRST>
__global__ __launch_bounds__(256) void sort_place_kernel(Tokens T, const Pair* __restrict__ in, SortMeta* meta,
                                                         SortPlan P, int shift, const uint32_t* __restrict__ counts,
                                                         Pair* __restrict__ out, uint8_t* __restrict__ used) {
    __shared__ uint32_t next[4][512];   // the wave's next free place of each digit
    __shared__ uint32_t total[512], scan[256];
    const int digits = 1 << P.bits, mask = digits - 1;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t count = FIRST ? T.positions : (int64_t)meta->valid;
    const int64_t lo = blockIdx.x * P.chunk, quarter = P.chunk / 4;
    const int64_t w_lo = lo + wave * quarter;
    int64_t w_hi = w_lo + quarter < count ? w_lo + quarter : count;
    for (int d = threadIdx.x; d < digits; d += 256)
#pragma unroll
        for (int w = 0; w < 4; ++w) next[w][d] = 0;
    __syncthreads();
    for (int64_t i = w_lo + lane; i < w_hi; i += 64) {
        Pair p;
        if (sort_item<IDX, FIRST>(T, in, i, w_hi, &p)) atomicAdd(&next[wave][(p.key >> shift) & mask], 1u);
    }
    // positions of this digit in the blocks before this one, and in all blocks
    uint32_t before[2] = {0, 0};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int d = threadIdx.x + h * 256;
        if (d >= digits) continue;
        uint32_t all = 0;
#pragma unroll 8
        for (int b = 0; b < P.blocks; ++b) {
            const uint32_t c = counts[(int64_t)b * digits + d];
            if (b < (int)blockIdx.x) before[h] += c;
            all += c;
        }
        total[d] = all;
    }
    __syncthreads();
    // exclusive sums over the digits: two digits per thread (d and d + 1 next to each other)
    uint32_t pair_sum = 0;
    if (2 * (int)threadIdx.x < digits) pair_sum = total[2 * threadIdx.x] + (2 * (int)threadIdx.x + 1 < digits ? total[2 * threadIdx.x + 1] : 0);
    scan[threadIdx.x] = pair_sum;
    __syncthreads();
    for (int o = 1; o < 256; o <<= 1) {
        const uint32_t x = (int)threadIdx.x >= o ? scan[threadIdx.x - o] : 0;
        __syncthreads();
        scan[threadIdx.x] += x;
        __syncthreads();
    }
    if (FIRST && blockIdx.x == 0 && threadIdx.x == 255) meta->valid = scan[255];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int d = threadIdx.x + h * 256;
        if (d >= digits) continue;
        const uint32_t upto = scan[d >> 1];   // through digit d | 1
        uint32_t at = upto - total[d] - ((d & 1) == 0 && d + 1 < digits ? total[d + 1] : 0) + before[h];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const uint32_t c = next[w][d];
            next[w][d] = at;
            at += c;
        }
    }
    __syncthreads();
    for (int64_t i0 = w_lo; i0 < w_hi; i0 += 64) {
        Pair p;
        const bool ok = sort_item<IDX, FIRST>(T, in, i0 + lane, w_hi, &p);
        const uint32_t digit = ok ? (p.key >> shift) & mask : 0;
        uint64_t peers = __ballot(ok);
        for (int b = 0; b < P.bits; ++b) {
            const bool bit = (digit >> b) & 1;
            const uint64_t ones = __ballot(bit);
            peers &= bit ? ones : ~ones;
        }
        if (ok) {
            const uint64_t below = peers & ((1ull << lane) - 1);
            const uint32_t first = next[wave][digit];
            out[first + __popcll(below)] = p;
            if (FIRST) used[p.key] = 1;   // every writer stores the same value
            if ((peers >> lane) == 1) next[wave][digit] = first + __popcll(peers);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the next step reads what this one moved on
    }
}

// ---- gradient: the sums ---------------------------------------------------------------------------
// A worker (one thread per chunk of EPV columns) walks `run` sorted positions and adds their rows while
// the key stays the same.  A run of one key inside the worker's range is a finished table row; a run that
// reaches over an end of the range leaves a partial sum: slot 0 what began before the range, slot 1 what
// goes on behind it.  The workgroups behind the workers clear the table rows no valid position holds.
struct SumPlan {
    int run;            // sorted positions per worker
    int cpr, rpp;       // chunks per row, workers side by side in a workgroup
    int64_t workers;    // over the largest possible number of valid positions
    int64_t sum_groups; // workgroups of workers; the rest clear rows
    int64_t pad_dim;    // floats of a partial row
};

template <typename OT, int EPV>
__device__ __forceinline__ void put_row(OT* table, int64_t key, int dim, int c, const float* acc, float scale) {
    Vec<OT, EPV> w;
#pragma unroll
    for (int e = 0; e < EPV; ++e) w.x[e] = from_f32<OT>(scale * acc[e]);
    store_vec<OT, EPV>(table + key * dim + (int64_t)c * EPV, w);
}

template <typename GT, typename OT, int EPV>
__global__ __launch_bounds__(256) void grad_sum_kernel(const GT* __restrict__ grad, const Pair* __restrict__ sorted,
                                                       const SortMeta* __restrict__ meta,
                                                       const uint8_t* __restrict__ used, int64_t vocab, float scale,
                                                       OT* __restrict__ table, int dim, SumPlan S,
                                                       float* __restrict__ partial, int32_t* __restrict__ chain_end) {
    const int r = S.cpr < 256 ? (int)threadIdx.x / S.cpr : 0;
    const int c0 = S.cpr < 256 ? (int)threadIdx.x - r * S.cpr : (int)threadIdx.x;
    if (r >= S.rpp) return;
    if ((int64_t)blockIdx.x >= S.sum_groups) {
        const float zero[EPV] = {};
        for (int64_t v = ((int64_t)blockIdx.x - S.sum_groups) * S.rpp + r; v < vocab;
             v += ((int64_t)gridDim.x - S.sum_groups) * S.rpp)
            if (!used[v])
                for (int c = c0; c < S.cpr; c += 256) put_row<OT, EPV>(table, v, dim, c, zero, 1.0f);
        return;
    }
    constexpr int U = 8;
    const int64_t valid = meta->valid;
    const int64_t worker = (int64_t)blockIdx.x * S.rpp + r;
    const int64_t lo = worker * S.run, hi = lo + S.run < valid ? lo + S.run : valid;
    if (lo >= hi) return;
    const bool head = lo > 0 && sorted[lo - 1].key == sorted[lo].key;
    const bool tail = hi < valid && sorted[hi].key == sorted[hi - 1].key;
    for (int c = c0; c < S.cpr; c += 256) {
        float acc[EPV] = {};
        uint32_t cur = sorted[lo].key;
        bool first = true;   // the run that opens the range
        auto flush = [&](bool last) {
            if ((first && head) || (last && tail)) {
                float* dst = partial + (worker * 2 + (first && head ? 0 : 1)) * S.pad_dim + (int64_t)c * EPV;
#pragma unroll
                for (int e = 0; e < EPV; ++e) dst[e] = acc[e];
                if (c == 0 && first && head && !(last && tail)) chain_end[cur] = (int32_t)worker;
            } else {
                put_row<OT, EPV>(table, cur, dim, c, acc, scale);
            }
        };
        for (int64_t i = lo; i < hi; i += U) {
            Pair p[U];
            Vec<GT, EPV> g[U];
#pragma unroll
            for (int u = 0; u < U; ++u) p[u] = sorted[i + u < hi ? i + u : hi - 1];
#pragma unroll
            for (int u = 0; u < U; ++u) g[u] = load_vec_nt<GT, EPV>(grad + (int64_t)p[u].pos * dim + (int64_t)c * EPV);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (i + u >= hi) break;
                if (p[u].key != cur) {
                    flush(false);
                    first = false;
                    cur = p[u].key;
#pragma unroll
                    for (int e = 0; e < EPV; ++e) acc[e] = 0.0f;
                }
#pragma unroll
                for (int e = 0; e < EPV; ++e) acc[e] += to_f32(g[u].x[e]);
            }
        }
        flush(true);
    }
}

// The runs that cross workers: the worker a run starts in is followed by partial sums of slot 0 up to
// chain_end.  A workgroup adds 64 columns of one run: 16 threads of 4 columns, 16 rows of partial sums side
// by side, joined in a fixed order.
template <typename OT>
__global__ __launch_bounds__(256) void grad_join_kernel(const Pair* __restrict__ sorted,
                                                        const SortMeta* __restrict__ meta, float scale,
                                                        OT* __restrict__ table, int dim, SumPlan S,
                                                        const float* __restrict__ partial,
                                                        const int32_t* __restrict__ chain_end) {
    __shared__ float part[16][64];
    const int64_t valid = meta->valid;
    const int col = blockIdx.y * 64 + (threadIdx.x & 15) * 4, lane = threadIdx.x >> 4;
    for (int64_t w = blockIdx.x; (w + 1) * S.run < valid; w += gridDim.x) {
        const int64_t lo = w * S.run, hi = lo + S.run;
        const uint32_t key = sorted[hi - 1].key;
        if (sorted[hi].key != key) continue;                                             // ends here
        if (sorted[lo].key == key && lo > 0 && sorted[lo - 1].key == key) continue;      // did not start here
        const int64_t n = chain_end[key] - w + 1;
        float acc[4] = {0, 0, 0, 0};
        if (col < (int)S.pad_dim)
            for (int64_t i = lane; i < n; i += 16) {
                const float4 x = *(const float4*)(partial + ((w + i) * 2 + (i == 0 ? 1 : 0)) * S.pad_dim + col);
                acc[0] += x.x;
                acc[1] += x.y;
                acc[2] += x.z;
                acc[3] += x.w;
            }
        *(float4*)&part[lane][(threadIdx.x & 15) * 4] = make_float4(acc[0], acc[1], acc[2], acc[3]);
        __syncthreads();
        if (threadIdx.x < 64) {
            const int c = blockIdx.y * 64 + threadIdx.x;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) sum += part[i][threadIdx.x];
            if (c < dim) table[(int64_t)key * dim + c] = from_f32<OT>(scale * sum);
        }
        __syncthreads();
    }
}
