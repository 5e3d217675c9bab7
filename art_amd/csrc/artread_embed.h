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
// of U rows; `cpr` chunks make a row, a workgroup holds `rpp` rows side by side.  The keys of its rows are
// requested before any table row, those before any store.  The U rows are a whole grid apart, so that the chip
// writes one window of consecutive rows at a time: with rows of a workgroup next to each other, U decided how
// many workgroups met on a memory channel (2,048 x 256 tokens of 768 bf16: U 1 246 us, 3 141, 8 215, 16 378);
// with them apart 149 us for U 2 and 4.  The table is read through the caches (a few thousand rows serve a whole
// batch), the output, which another kernel reads much later, is stored past them (251-340 us if it is not).
// Bound by those stores: 147 us for 0.8 GB of them, 5.5 TB/s.
constexpr int kEmbedRows = 2;
template <typename TT, typename OT, typename IDX, int EPV>
__global__ __launch_bounds__(256) void embed_kernel(const TT* __restrict__ table, int64_t table_stride, Tokens T,
                                                    float scale, OT* __restrict__ out, int dim, int cpr, int rpp) {
    constexpr int U = kEmbedRows;
    const int r = cpr < 256 ? (int)threadIdx.x / cpr : 0;
    const int c0 = cpr < 256 ? (int)threadIdx.x - r * cpr : (int)threadIdx.x;
    if (r >= rpp) return;
    const int64_t apart = (int64_t)gridDim.x * rpp;
    for (int64_t base = (int64_t)blockIdx.x * rpp + r; base < T.positions; base += apart * U) {
        int32_t key[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t pos = base + u * apart;
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
                const int64_t pos = base + u * apart;
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
// workgroup's chunk, then each workgroup derives its own bases from all counts and places its chunk.  Up to
// kSortAlone positions are one workgroup's, which makes all passes in one launch.  What a pass costs is the
// length of its chains (steps of a wave, rows of counts), not its bytes: hence sixteen waves a workgroup.  2,048 x 256
// positions: counts 5 us and places 11 us a pass, of which there are two; 67 x 61 in one workgroup: 14 us.
constexpr int kSortThreads = 1024, kSortWaves = 16, kSortDigits = 512;
constexpr int64_t kSortAlone = 16384;
struct SortPlan {
    int blocks;       // chunks of the position list
    int64_t chunk;    // positions per chunk, a multiple of kSortThreads
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

// digit counts [blocks][1 << bits]
template <typename IDX, bool FIRST>
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(Tokens T, const Pair* __restrict__ in,
                                                                  const SortMeta* __restrict__ meta, SortPlan P,
                                                                  int shift, uint32_t* __restrict__ counts) {
    __shared__ uint32_t hist[kSortDigits];
    const int digits = 1 << P.bits;
    if ((int)threadIdx.x < digits) hist[threadIdx.x] = 0;
    __syncthreads();
    const int64_t count = FIRST ? T.positions : (int64_t)meta->valid;
    const int64_t lo = blockIdx.x * P.chunk, hi = lo + P.chunk < count ? lo + P.chunk : count;
    for (int64_t i = lo + threadIdx.x; i < hi; i += kSortThreads) {
        Pair p;
        if (sort_item<IDX, FIRST>(T, in, i, hi, &p)) atomicAdd(&hist[(p.key >> shift) & (digits - 1)], 1u);
    }
    __syncthreads();
    if ((int)threadIdx.x < digits) counts[(int64_t)blockIdx.x * digits + threadIdx.x] = hist[threadIdx.x];
}

struct SortSpace {
    uint32_t next[kSortWaves][kSortDigits];   // a wave's next free place of each digit
    uint32_t total[kSortDigits], before[kSortDigits], scan[kSortDigits];
};

// Places one chunk.  Each wave owns a part of it and walks the part in order, 64 positions at a time: the lanes
// that share a digit find each other by `bits` ballots, the lane's rank is the number of them below it, and the
// highest one moves the wave's next free place of that digit on.  counts: of all chunks, nullptr where this is the
// only one.  Returns the number of positions placed by all chunks.
template <typename IDX, bool FIRST>
__device__ __forceinline__ uint32_t sort_place(const Tokens& T, const Pair* in, int64_t count, const SortPlan& P,
                                               int shift, const uint32_t* counts, Pair* out, SortSpace& S) {
    const int digits = 1 << P.bits, mask = digits - 1;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t part = P.chunk / kSortWaves, w_lo = blockIdx.x * P.chunk + wave * part;
    const int64_t w_hi = w_lo + part < count ? w_lo + part : count;
    for (int i = threadIdx.x; i < kSortWaves * kSortDigits; i += kSortThreads) (&S.next[0][0])[i] = 0;
    if (threadIdx.x < kSortDigits) S.total[threadIdx.x] = S.before[threadIdx.x] = 0;
    __syncthreads();
    for (int64_t i = w_lo + lane; i < w_hi; i += 64) {
        Pair p;
        if (sort_item<IDX, FIRST>(T, in, i, w_hi, &p)) atomicAdd(&S.next[wave][(p.key >> shift) & mask], 1u);
    }
    if (counts) {   // positions of each digit in all chunks, and in those before this one; several threads a digit
        const int d = threadIdx.x & mask, each = kSortThreads >> P.bits, mine = threadIdx.x >> P.bits;
        uint32_t all = 0, ahead = 0;
#pragma unroll 8
        for (int b = mine; b < P.blocks; b += each) {
            const uint32_t c = counts[(int64_t)b * digits + d];
            if (b < (int)blockIdx.x) ahead += c;
            all += c;
        }
        atomicAdd(&S.total[d], all);
        atomicAdd(&S.before[d], ahead);
    }
    __syncthreads();
    if (!counts && (int)threadIdx.x < digits) {
        uint32_t all = 0;
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) all += S.next[w][threadIdx.x];
        S.total[threadIdx.x] = all;
    }
    __syncthreads();
    if (threadIdx.x < kSortDigits) {   // inclusive sums over the digits, by wave
        uint32_t x = S.total[threadIdx.x];
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t y = __shfl_up(x, o);
            if (lane >= o) x += y;
        }
        S.scan[threadIdx.x] = x;
    }
    __syncthreads();
    uint32_t lower = 0;
    if (threadIdx.x < kSortDigits)
        for (int w = 0; w < wave; ++w) lower += S.scan[64 * w + 63];
    __syncthreads();
    if (threadIdx.x < kSortDigits) S.scan[threadIdx.x] += lower;
    __syncthreads();
    if ((int)threadIdx.x < digits) {
        uint32_t at = S.scan[threadIdx.x] - S.total[threadIdx.x] + S.before[threadIdx.x];
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) {
            const uint32_t c = S.next[w][threadIdx.x];
            S.next[w][threadIdx.x] = at;
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
            const uint32_t first = S.next[wave][digit];
            out[first + __popcll(below)] = p;
            if ((peers >> lane) == 1) S.next[wave][digit] = first + __popcll(peers);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the next step reads what this one moved on
    }
    return S.scan[digits - 1];
}

template <typename IDX, bool FIRST>
__global__ __launch_bounds__(kSortThreads) void sort_place_kernel(Tokens T, const Pair* __restrict__ in, SortMeta* meta,
                                                                  SortPlan P, int shift,
                                                                  const uint32_t* __restrict__ counts,
                                                                  Pair* __restrict__ out) {
    __shared__ SortSpace S;
    const int64_t count = FIRST ? T.positions : (int64_t)meta->valid;
    const uint32_t placed = sort_place<IDX, FIRST>(T, in, count, P, shift, counts, out, S);
    if (FIRST && blockIdx.x == 0 && threadIdx.x == 0) meta->valid = placed;
}

// all passes of a list that one workgroup takes; the result lies in a or b as sort_tokens says
template <typename IDX>
__global__ __launch_bounds__(kSortThreads) void sort_alone_kernel(Tokens T, SortMeta* meta, SortPlan P, Pair* a, Pair* b) {
    __shared__ SortSpace S;
    const int64_t valid = sort_place<IDX, true>(T, nullptr, T.positions, P, 0, nullptr, a, S);
    if (threadIdx.x == 0) meta->valid = (uint32_t)valid;
    for (int pass = 1; pass < P.passes; ++pass) {
        __syncthreads();   // the pairs are written: the workgroup shares its cache
        sort_place<IDX, false>(T, pass & 1 ? a : b, valid, P, pass * P.bits, nullptr, pass & 1 ? b : a, S);
    }
}

// ---- gradient: the sums ---------------------------------------------------------------------------
// A worker (one thread per chunk of EPV columns) walks a range of `run` sorted positions and adds their rows while
// the key stays the same.  A run of one key inside the range is a finished table row; a run that reaches over an
// end of the range leaves a partial sum: slot 0 what began before the range, slot 1 what goes on behind it.  The
// workgroups behind the workers clear the table rows that no valid position holds.  Bound by reading the gradient
// and writing the table: 113 us for 2,048 x 256 positions of 768 f16, 62 % valid, 4.9 TB/s.  (Workers that read on
// behind their range to finish a run there leave only the longest runs to the join, but are up to twice as long
// themselves: 154 us.)
struct SumPlan {
    int run;            // sorted positions of a range
    int cpr, rpp;       // chunks per row, workers side by side in a workgroup
    int64_t workers;    // over the largest possible number of valid positions
    int64_t sum_groups; // workgroups of workers; the rest clear rows
    int64_t pad_dim;    // floats of a partial row
};
constexpr int kClearRows = 64;   // table rows of a clearing workgroup: a lane of each looks for its row

template <typename OT, int EPV>
__device__ __forceinline__ void put_row(OT* table, int64_t key, int dim, int c, const float* acc, float scale) {
    Vec<OT, EPV> w;
#pragma unroll
    for (int e = 0; e < EPV; ++e) w.x[e] = from_f32<OT>(scale * acc[e]);
    store_vec<OT, EPV>(table + key * dim + (int64_t)c * EPV, w);
}

template <typename GT, typename OT, int EPV>
__global__ __launch_bounds__(256) void grad_sum_kernel(const GT* __restrict__ grad, const Pair* __restrict__ sorted,
                                                       const SortMeta* __restrict__ meta, int64_t vocab, float scale,
                                                       OT* __restrict__ table, int dim, SumPlan S,
                                                       float* __restrict__ partial, int32_t* __restrict__ chain_end) {
    const int64_t valid = meta->valid;
    if ((int64_t)blockIdx.x >= S.sum_groups) {
        __shared__ uint64_t empty_rows;
        const float zero[EPV] = {};
        for (int64_t v0 = ((int64_t)blockIdx.x - S.sum_groups) * kClearRows; v0 < vocab;
             v0 += ((int64_t)gridDim.x - S.sum_groups) * kClearRows) {
            if (threadIdx.x < 64) {
                const int64_t v = v0 + threadIdx.x;
                int64_t lo = 0, hi = valid;   // the first position whose key is not below v
                while (lo < hi) {
                    const int64_t mid = (lo + hi) >> 1;
                    if ((int64_t)sorted[mid].key < v) lo = mid + 1;
                    else hi = mid;
                }
                const uint64_t found = __ballot(v < vocab && (lo >= valid || (int64_t)sorted[lo].key != v));
                if (threadIdx.x == 0) empty_rows = found;
            }
            __syncthreads();
            for (uint64_t rows = empty_rows; rows; rows &= rows - 1)
                for (int c = threadIdx.x; c < S.cpr; c += blockDim.x)
                    put_row<OT, EPV>(table, v0 + __ffsll((unsigned long long)rows) - 1, dim, c, zero, 1.0f);
            __syncthreads();
        }
        return;
    }
    const int r = S.cpr < 256 ? (int)threadIdx.x / S.cpr : 0;
    const int c0 = S.cpr < 256 ? (int)threadIdx.x - r * S.cpr : (int)threadIdx.x;
    if (r >= S.rpp) return;
    constexpr int U = 8;
    const int64_t worker = (int64_t)blockIdx.x * S.rpp + r;
    const int64_t lo = worker * S.run, hi = lo + S.run < valid ? lo + S.run : valid;
    if (lo >= hi) return;
    const uint32_t first_key = sorted[lo].key;
    const bool head = lo > 0 && sorted[lo - 1].key == first_key;
    const bool tail = hi < valid && sorted[hi].key == sorted[hi - 1].key;
    for (int c = c0; c < S.cpr; c += 256) {
        float acc[EPV] = {};
        uint32_t cur = first_key;
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

// The runs that cross ranges: the range one begins in is followed by partial sums of slot 0 up to chain_end.  A
// workgroup of sixteen waves takes sixteen ranges and 256 columns.  A run of up to kJoinShort partial sums is its
// range's wave's; the longer ones are added by all waves, each every sixteenth partial sum, joined in order: 12 us at
// 2,048 x 256 positions, the chain of the longest run.
constexpr int kJoinWaves = 16, kJoinShort = 16;
template <typename OT>
__global__ __launch_bounds__(64 * kJoinWaves) void grad_join_kernel(const Pair* __restrict__ sorted,
                                                                    const SortMeta* __restrict__ meta, float scale,
                                                                    OT* __restrict__ table, int dim, SumPlan S,
                                                                    const float* __restrict__ partial,
                                                                    const int32_t* __restrict__ chain_end) {
    __shared__ float4 part[kJoinWaves][64];
    __shared__ int longs[kJoinWaves];   // partial sums of a long run that begins in the wave's range
    const int64_t valid = meta->valid, w0 = (int64_t)blockIdx.x * kJoinWaves;
    if ((w0 + 1) * S.run >= valid) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = (blockIdx.y * 64 + lane) * 4;
    auto add = [&](int64_t w, int64_t i0, int64_t n, int64_t step) {
        float4 acc = make_float4(0, 0, 0, 0);
        if (col < (int)S.pad_dim) {
#pragma unroll 4
            for (int64_t i = i0; i < n; i += step) {
                const float4 x = *(const float4*)(partial + ((w + i) * 2 + (i == 0 ? 1 : 0)) * S.pad_dim + col);
                acc.x += x.x;
                acc.y += x.y;
                acc.z += x.z;
                acc.w += x.w;
            }
        }
        return acc;
    };
    auto put = [&](uint32_t key, const float4& sum) {
        const float y[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < dim) table[(int64_t)key * dim + col + e] = from_f32<OT>(scale * y[e]);
    };
    {
        const int64_t w = w0 + wave, lo = w * S.run, hi = lo + S.run;
        int64_t n = 0;
        uint32_t key = 0;
        if (hi < valid) {
            key = sorted[hi - 1].key;
            const bool began = lo > 0 && sorted[lo].key == key && sorted[lo - 1].key == key;
            if (sorted[hi].key == key && !began) n = chain_end[key] - w + 1;
        }
        if (n > 0 && n <= kJoinShort) put(key, add(w, 0, n, 1));
        if (lane == 0) longs[wave] = n > kJoinShort ? (int)n : 0;
    }
    __syncthreads();
    for (int x = 0; x < kJoinWaves; ++x) {
        const int n = longs[x];
        if (!n) continue;
        part[wave][lane] = add(w0 + x, wave, n, kJoinWaves);
        __syncthreads();
        if (wave == 0) {
            float4 sum = part[0][lane];
#pragma unroll
            for (int i = 1; i < kJoinWaves; ++i) {
                const float4 y = part[i][lane];
                sum.x += y.x;
                sum.y += y.y;
                sum.z += y.z;
                sum.w += y.w;
            }
            put(sorted[(w0 + x + 1) * S.run - 1].key, sum);
        }
        __syncthreads();
    }
}
