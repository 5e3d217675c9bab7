// Attention of query rows to the states of their passages, and its gradient (include/artread.h).
// Included by artread.hip only.
//
// The rows of one batch entry that read one key head (rows x the heads that share it) are numbered r, query
// position major; a workgroup or wave takes a block of them.  All products are 32x32x16 MFMAs:
//   lane l of A holds row l & 31, of B column l & 31, both 8 consecutive k at 8 * (l >> 5);
//   lane l of C holds column l & 31 and, in element i, row 8 * (i >> 2) + 4 * (l >> 5) + (i & 3).
// Scores are computed as S^T = K Q^T, so a lane owns one query row and the softmax of a row is arithmetic
// inside two lanes.  The weights P^T then lie where the next product wants its B operand, if its k index runs
// over the keys in C's order; V^T as the A operand follows that order through the transposing LDS read
// (ds_read_b64_tr_b16: four rows of the tile as four consecutive k).  So no weight ever crosses lanes.
#pragma once
#include <type_traits>

#include "artread_common.h"

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Mma;
template <>
struct Mma<f16> {
    typedef f16 V8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x16 mul(V8 a, V8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    // Weights of a softmax keep 2^10 beside them while they are f16: the smallest normal f16 is 2^-14, so a weight
    // of one key among tens of thousands would else lose bits.  Sums carry the same factor, and it cancels.
    static constexpr float kWeightLog2 = 10.0f;
    static constexpr float kSlack = 5.0f;   // weights reach 2^15
};
template <>
struct Mma<bf16> {
    typedef bf16 V8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x16 mul(V8 a, V8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
    static constexpr float kWeightLog2 = 0.0f;   // the exponent of f32
    static constexpr float kSlack = 8.0f;
};

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// ---- the problem as the kernels see it --------------------------------------------------------------
struct AttendPlan {
    int64_t row_count;    // rows x share
    int64_t pad_rows;     // row_count in whole tiles of 64: the gradient's row statistics
    int64_t row_blocks;   // blocks of rows per (batch entry, key head)
    int64_t items;        // batch x kv_heads x row_blocks
    uint32_t pack, inv_pack;     // entries of a passage where short passages are packed, 0 where not; floor(2^32 / pack)
    int64_t pack_passages;       // passages of a batch entry there; the problem then has one, pack_passages x pack long
    uint32_t share, inv_share;   // heads per key head; floor(2^32 / share), 2^32 - 1 for 1
    int walkers;          // waves of a workgroup that walk one item
    int splits;           // parts the keys of an item are dealt to
    int by_head;          // order of the key walk's items
    float c;              // |scale| * log2(e)
    float unweight;       // takes back the factor that f16 weights carry
    uint32_t q_and, q_xor;   // scale's sign (and zero) applied to the bits of q: c stays positive
};

// Grids are two-dimensional, so that one workgroup an item never meets a grid's limits.
__device__ __forceinline__ int64_t block_id() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

// query position and head of row r < 2^31: the quotient from inv_share is at most one too small
__device__ __forceinline__ void split_row(const AttendPlan& P, int64_t kh, uint32_t r, int64_t* t, int64_t* h) {
    uint32_t q = __umulhi(r, P.inv_share), g = r - q * P.share;
    if (g >= P.share) {
        q += 1;
        g -= P.share;
    }
    *t = q;
    *h = kh * P.share + g;
}

// Valid entries of a packed batch entry from entry f0 on, one per lane: the lane's passage's length is asked for here
// and compared when it is needed.
struct Packed {
    const int32_t* lengths;   // of the batch entry
    uint32_t pack, inv_pack;
    int total;                // entries
    int entry, length;        // the lane's, in its passage; the passage's length
    __device__ __forceinline__ void start(const artread_attend_t& A, const AttendPlan& P, int64_t b) {
        lengths = A.lengths + b * P.pack_passages;
        pack = P.pack;
        inv_pack = P.inv_pack;
        total = (int)A.len;
    }
    __device__ __forceinline__ void ask(int f) {
        entry = length = 0;
        if (f < total) {
            uint32_t p = __umulhi((uint32_t)f, inv_pack), j = (uint32_t)f - p * pack;
            if (j >= pack) {   // the quotient is at most one too small
                p += 1;
                j -= pack;
            }
            entry = (int)j;
            length = lengths[p];
        }
    }
    __device__ __forceinline__ bool valid() const { return entry < length; }
};

// Deals the tiles of KT keys of a batch entry's passages to `splits` walkers, one after the other; a passage's
// last tile may be short, the next passage starts a new tile.  Lengths are held 64 passages at a time, one per
// lane, beside the number of tiles up to each, so that a tile is found at once however many passages lie between (walking
// over them one by one took 187 us of 1,000 passages of 40, dealt to 32).  Passages too short to fill tiles of their own
// are packed: the batch entry is one long passage with holes.  Either way `mask` says which of a tile's keys are valid.
// All of it is uniform over the wave.
template <int KT>
struct Walk {
    const int32_t* lengths;
    Packed packed;
    uint64_t mask;
    int passages, len, p, n, j0, step;
    int chunk, tile, tiles, splits;   // first passage held; the tile among those held, which are `tiles`
    int held, upto;                   // the lane's passage's length, and the tiles up to and with it
    bool is_packed, moved;            // moved: to another passage, or from nowhere
    __device__ __forceinline__ void hold() {
        const int lane = threadIdx.x & 63, i = chunk + lane;
        int x = i < passages ? len : 0;
        if (lengths && i < passages) x = lengths[i];
        held = x < 0 ? 0 : (x < len ? x : len);
        upto = (held + KT - 1) / KT;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(upto, o);
            if (lane >= o) upto += y;
        }
        tiles = __builtin_amdgcn_readlane(upto, 63);
    }
    __device__ __forceinline__ void start(const artread_attend_t& A, const AttendPlan& P, int64_t b, int split, int of) {
        is_packed = P.pack != 0;
        passages = (int)A.passages;
        len = (int)A.len;
        splits = of;
        step = splits * KT;
        moved = true;   // a packed entry's only passage is told once
        if (is_packed) {
            lengths = nullptr;
            p = 0;
            j0 = split * KT;
            packed.start(A, P, b);
            packed.ask(j0 + (int)(threadIdx.x & 63));
        } else {
            lengths = A.lengths ? A.lengths + b * A.passages : nullptr;
            p = j0 = n = chunk = 0;
            tile = split;
            hold();
        }
    }
    // false: no tile left; else passage p, first key j0, and mask
    __device__ __forceinline__ bool settle() {
        if (is_packed) {
            if (j0 >= len) return false;
            mask = __ballot(packed.valid());
            return true;
        }
        if (j0 >= n) {
            while (tile >= tiles) {
                tile -= tiles;
                chunk += 64;
                if (chunk >= passages) return false;
                hold();
            }
            const int l = __ffsll((unsigned long long)__ballot(upto > tile)) - 1;
            n = __builtin_amdgcn_readlane(held, l);
            j0 = (tile - __builtin_amdgcn_readlane(upto, l)) * KT + (n + KT - 1) / KT * KT;
            p = chunk + l;
            moved = true;
        }
        const int left = n - j0;
        mask = left >= 64 ? ~0ull : (1ull << left) - 1;
        return true;
    }
    __device__ __forceinline__ void advance() {
        moved = false;
        tile += splits;
        j0 += step;
        if (is_packed) packed.ask(j0 + (int)(threadIdx.x & 63));   // in time for the tile after this one
    }
};
template <int KB>
__device__ __forceinline__ bool whole_tile(uint64_t mask) { return KB == 1 ? (uint32_t)mask == ~0u : mask == ~0ull; }

// 16-byte pieces of rows: zero behind `dim` and for rows that are not there
template <typename T>
__device__ __forceinline__ typename Mma<T>::V8 load8(const T* p, bool ok) {
    typename Mma<T>::V8 v = {};
    if (ok) v = *(const typename Mma<T>::V8*)p;
    return v;
}

// ---- LDS tiles of DP columns --------------------------------------------------------------------------
// 16-byte chunks of a row are permuted by the row's number, so that both ways of reading meet every bank once: 16
// rows of one chunk (A operands of rows), and the four rows x 64 bytes of half a wave's transposing read.
template <int DP>
__device__ __forceinline__ int tile_chunk(int row, int chunk) {
    return DP == 128 ? chunk ^ (((row & 3) << 2) | ((row >> 2) & 3)) : chunk ^ ((((row >> 1) & 1) << 2) | ((row >> 2) & 3));
}
// The permutation only flips address bits below a row's size, so a lane's addresses differ from one base by XORs
// with constants: one register for each way of reading a tile.  `opaque` keeps the compiler from holding all of them.
__device__ __forceinline__ uint32_t lds_offset(const void* p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}
__device__ __forceinline__ uint32_t opaque(uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
}
// a lane's place in the first row block of a tile, read as rows
template <int DP>
__device__ __forceinline__ uint32_t rows_base(int lane) {
    const int row = lane & 31;
    return (uint32_t)(row * DP * 2 + tile_chunk<DP>(row, lane >> 5) * 16);
}
// A operand: rows 32 * block + (l & 31), columns 16 * s + 8 * (l >> 5)..
template <typename T, int DP>
__device__ __forceinline__ typename Mma<T>::V8 lds_rows(uint32_t base, int block, int s) {
    typedef const __attribute__((address_space(3))) typename Mma<T>::V8* P;
    return *(P)(uintptr_t)((base ^ (uint32_t)(32 * s)) + (uint32_t)(block * 32 * DP * 2));
}
// a lane's place in the first 16 rows of a tile, read as columns
template <int DP>
__device__ __forceinline__ uint32_t columns_base(int lane) {
    const int i = lane & 15, row = 4 * (lane >> 5) + (i >> 2), col = (lane & 16) + 4 * (i & 3);
    return (uint32_t)(row * DP * 2 + tile_chunk<DP>(row, col >> 3) * 16 + (col & 7) * 2);
}
// A operand of the transposed tile: columns 32 * db + (l & 31), k over rows r0 + {4 half + 0..3, 8 + 4 half + 0..3};
// r0 is a multiple of 16
template <typename T, int DP>
__device__ __forceinline__ typename Mma<T>::V8 lds_columns(uint32_t base, int r0, int db) {
    union {
        s16x4 h[2];
        typename Mma<T>::V8 v;
    } u;
#pragma unroll
    for (int x = 0; x < 2; ++x)
        u.h[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(uintptr_t)(
            (base ^ (uint32_t)(64 * db + 32 * x)) + (uint32_t)((r0 + 8 * x) * DP * 2)));
    return u.v;
}

// ---- memory straight to LDS ---------------------------------------------------------------------------
// One wave-instruction moves 64 x 16 (or 64 x 4) bytes: lane i's piece lands at dst + 16 * i (4 * i), so the chunk
// order of the tile is made on the source side.  The compiler does not count these loads: dma_wait<N> waits until at
// most N of the wave's vector memory operations are outstanding (its own only make that stricter).
// Sources are a uniform base plus 32 bits of bytes per lane.
__device__ __forceinline__ const void* uniform_ptr(const void* p) {
    const uint64_t u = (uint64_t)(uintptr_t)p;
    const uint64_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)u);
    const uint64_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(u >> 32));
    return (const void*)(uintptr_t)(lo | hi << 32);
}
__device__ __forceinline__ void dma16(const void* base, uint32_t lane_bytes, uint32_t dst) {
    uint32_t keep;
    asm volatile("s_nop 4\n\ts_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %2\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "s"(dst), "s"(uniform_ptr(base)), "v"(lane_bytes) : "memory");
}
// N pieces `step` bytes apart in memory and STEP in LDS, those of piece x from lane offsets off[x]
template <int N, int STEP>
__device__ __forceinline__ void dma_pieces(const void* base, uint32_t step, const uint32_t* off, uint32_t dst) {
    static_assert(N == 1 || N == 2 || N == 4, "");
    const char* at = (const char*)uniform_ptr(base);
    uint32_t keep;
    if constexpr (N == 1) {
        dma16(at, off[0], dst);
    } else if constexpr (N == 2) {
        asm volatile("s_nop 4\n\ts_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %5, %3\n\t"
                     "s_add_u32 m0, m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %6, %4\n\ts_mov_b32 m0, %0"
                     : "=&s"(keep) : "s"(dst), "n"(STEP), "s"(at), "s"(at + step), "v"(off[0]), "v"(off[1]) : "memory", "scc");
    } else {
        asm volatile("s_nop 4\n\ts_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %7, %3\n\t"
                     "s_add_u32 m0, m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %8, %4\n\t"
                     "s_add_u32 m0, m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %9, %5\n\t"
                     "s_add_u32 m0, m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %10, %6\n\ts_mov_b32 m0, %0"
                     : "=&s"(keep) : "s"(dst), "n"(STEP), "s"(at), "s"(at + step), "s"(at + 2 * (uint64_t)step),
                       "s"(at + 3 * (uint64_t)step), "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]) : "memory", "scc");
    }
}
__device__ __forceinline__ void dma4(const void* base, uint32_t lane_bytes, uint32_t dst) {
    uint32_t keep;
    asm volatile("s_nop 4\n\ts_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %3, %2\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "s"(dst), "s"(uniform_ptr(base)), "v"(lane_bytes) : "memory");
}
// also every LDS read of the wave is done: the barrier behind it lets others refill what it read
template <int N>
__device__ __forceinline__ void dma_wait() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wave_meet() { asm volatile("s_barrier" ::: "memory"); }

// ---- softmax over one tile ----------------------------------------------------------------------------
// the two halves of a wave hold one column between them: the greater, and the sum, of their values for both
__device__ __forceinline__ float both_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float both_sum(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// scores of NB x 32 keys of one row per lane pair -> weights; m, l are the running maximum (of scores x c) and the
// lane's own part of the sum, `o` the accumulators that a new maximum rescales.  A row's maximum is followed once it is
// passed by a factor of 2^kSlack: among 32 rows nearly every tile has some new maximum, hardly any such a one (8 x 8 x
// 512 states of 128 columns, 4096 rows a key head: 282 us against 296).
template <typename T, int NB, int NO>
__device__ __forceinline__ void softmax_tile(f32x16 (&s)[NB], float c, uint64_t mask, int half, float& m, float& l,
                                             f32x16 (&o)[NO]) {
    if (!whole_tile<NB>(mask)) {
        const uint64_t mine = mask >> (4 * half);   // keys of this lane's rows of C
        asm volatile("");                           // a branch: most tiles are whole
#pragma unroll
        for (int kb = 0; kb < NB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (!((uint32_t)(mine >> (32 * kb)) & (1u << (8 * (i >> 2) + (i & 3))))) s[kb][i] = -INFINITY;
    }
    float top = s[0][0];
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[kb][i]);
    top = both_max(top) * c;
    if (__any(top > m + Mma<T>::kSlack)) {
        const float m1 = top > m + Mma<T>::kSlack ? top : m;   // by the row alone, whatever its neighbours hold
        const float f = m1 == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - m1);
        m = m1;
        l *= f;
#pragma unroll
        for (int x = 0; x < NO; ++x)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[x][i] *= f;
    }
    const float base = (m == -INFINITY ? 0.0f : m) - Mma<T>::kWeightLog2;
    float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};   // four chains instead of one as long as the tile
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[kb][i] = __builtin_amdgcn_exp2f(fmaf(s[kb][i], c, -base));
            part[i & 3] += s[kb][i];
        }
    l += (part[0] + part[1]) + (part[2] + part[3]);
}

template <typename T>
__device__ __forceinline__ typename Mma<T>::V8 weights8(const f32x16& s, int ks) {
    typename Mma<T>::V8 p;
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = (T)s[8 * ks + e];   // rounded once, to nearest
    return p;
}

// ---- what a block of rows leaves ----------------------------------------------------------------------
// One split: the rows themselves.  Several: accumulators, maximum and sum of every row for the join.
struct Partials {
    float* o;      // [splits][all rows][dim]
    float2* ml;    // [splits][all rows]
    int64_t rows;  // batch x kv_heads x row_count
};

template <typename T>
__device__ __forceinline__ void finish_row4(const artread_attend_t& A, int64_t at, int d, const float* o) {
    Vec<T, 4> w, e;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        w.x[x] = (T)o[x];
        e.x[x] = (T)(o[x] - (float)w.x[x]);
    }
    store_vec<T, 4>((T*)A.out + at + d, w);
    if (A.rest) store_vec<T, 4>((T*)A.rest + at + d, e);
}

__device__ __forceinline__ float log_sum(float m, float l, float weight_log2) {
    return l == 0.0f ? -INFINITY : (m - weight_log2) * kLn2 + logf(l);
}

template <typename T, int DP>
__device__ __forceinline__ void finish_rows(const artread_attend_t& A, const AttendPlan& P, const Partials& W, int64_t b,
                                            int64_t kh, int64_t r, int split, int half, float m, float l,
                                            f32x16 (&o)[DP / 32]) {
    if (r >= P.row_count) return;
    const int dim = (int)A.dim;
    if (P.splits > 1) {
        const int64_t at = split * W.rows + (b * A.kv_heads + kh) * P.row_count + r;
        if (half == 0) W.ml[at] = make_float2(m, l);
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int d = 32 * db + 8 * x + 4 * half;
                if (d < dim) *(float4*)(W.o + at * dim + d) = make_float4(o[db][4 * x], o[db][4 * x + 1], o[db][4 * x + 2], o[db][4 * x + 3]);
            }
        return;
    }
    int64_t t, h;
    split_row(P, kh, (uint32_t)r, &t, &h);
    const int64_t at = ((b * A.rows + t) * A.heads + h) * dim;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;   // no key: zeros
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int d = 32 * db + 8 * x + 4 * half;
            const float y[4] = {o[db][4 * x] * inv, o[db][4 * x + 1] * inv, o[db][4 * x + 2] * inv, o[db][4 * x + 3] * inv};
            if (d < dim) finish_row4<T>(A, at, d, y);
        }
    if (A.lse && half == 0) A.lse[(b * A.heads + h) * A.rows + t] = log_sum(m, l, Mma<T>::kWeightLog2);
}

// Joins the splits of a row: 32 lanes of four columns each, G groups of lanes that take every G-th split side by
// side.  G is 1 for a few splits (eight rows a workgroup) and 8 for many (one row a workgroup: the sum over 256
// splits is then 32 steps long).  The groups' sums are added in a fixed order.  Its bytes are few, so what it takes
// is a chain of dependent loads: 5 us for 768 rows of 64 columns in 2 splits, 6 us for 64 of 128 in 32, 9 us for 4,608
// of 64 in 8.
template <typename T, int G>
__global__ __launch_bounds__(256) void attend_join_kernel(artread_attend_t A, AttendPlan P, Partials W) {
    __shared__ float part[8][32][5];
    const int lane = threadIdx.x & 31, d = lane * 4, group = threadIdx.x >> 5;
    const int mine = G == 1 ? 0 : group;
    for (int64_t R0 = (int64_t)blockIdx.x * (8 / G); R0 < W.rows; R0 += (int64_t)gridDim.x * (8 / G)) {
        const int64_t R = G == 1 ? R0 + group : R0;
        const bool there = R < W.rows;
        float m = -INFINITY, l = 0.0f, o[4] = {0, 0, 0, 0};
        if (there) {
            for (int s = lane; s < P.splits; s += 32) m = fmaxf(m, W.ml[s * W.rows + R].x);
            for (int x = 16; x; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
            const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll 4
            for (int s = mine; s < P.splits; s += G) {
                const float2 ml = W.ml[s * W.rows + R];   // a split without keys: -inf, 0 and zeros
                const float f = exp2f(ml.x - base);
                l += f * ml.y;
                if (d < (int)A.dim) {
                    const float4 x = *(const float4*)(W.o + (s * W.rows + R) * A.dim + d);
                    o[0] += f * x.x;
                    o[1] += f * x.y;
                    o[2] += f * x.z;
                    o[3] += f * x.w;
                }
            }
        }
        if (G > 1) {
            part[group][lane][0] = l;
#pragma unroll
            for (int x = 0; x < 4; ++x) part[group][lane][1 + x] = o[x];
            __syncthreads();
            l = o[0] = o[1] = o[2] = o[3] = 0.0f;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                l += part[g][lane][0];
#pragma unroll
                for (int x = 0; x < 4; ++x) o[x] += part[g][lane][1 + x];
            }
            __syncthreads();
        }
        if (!there || (G > 1 && group != 0)) continue;
        const int64_t r = R % P.row_count, bk = R / P.row_count, kh = bk % A.kv_heads, b = bk / A.kv_heads;
        int64_t t, h;
        split_row(P, kh, (uint32_t)r, &t, &h);
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int x = 0; x < 4; ++x) o[x] *= inv;
        if (d < (int)A.dim) finish_row4<T>(A, ((b * A.rows + t) * A.heads + h) * A.dim, d, o);
        if (A.lse && lane == 0) A.lse[(b * A.heads + h) * A.rows + t] = log_sum(m, l, Mma<T>::kWeightLog2);
    }
}

// Q^T operand of a row block: row r, all columns, in registers for the whole walk
template <typename T, int DP>
__device__ __forceinline__ void load_q(const artread_attend_t& A, const AttendPlan& P, const T* base, int64_t s_batch,
                                       int64_t s_row, int64_t s_head, int64_t b, int64_t kh, int64_t r, int half,
                                       uint32_t q_and, uint32_t q_xor, typename Mma<T>::V8 (&q)[DP / 16]) {
    int64_t t, h;
    split_row(P, kh, (uint32_t)r, &t, &h);
    const T* src = base + b * s_batch + t * s_row + h * s_head;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        const int d = 16 * s + 8 * half;
        union {
            typename Mma<T>::V8 v;
            uint32_t u[4];
        } x;
        x.v = load8<T>(src + d, r < P.row_count && d < (int)A.dim);
#pragma unroll
        for (int e = 0; e < 4; ++e) x.u[e] = (x.u[e] & q_and) ^ q_xor;
        q[s] = x.v;
    }
}

// ---- few rows: one wave walks its tiles alone ----------------------------------------------------------
// QB x 32 rows per wave, 32 keys per tile.  Every key and value is read once, so this is bound by HBM: K goes
// straight from memory into the A operand, V through a tile of LDS of the wave's own for the transposing read,
// the next tile's loads are in flight while this one is worked on, and no wave waits for another.  Where items are
// few, the four waves of a workgroup walk one item between them (P.walkers of 4) and join what they have in LDS,
// so that a quarter of the partial results is left to the join kernel, or none.
//   64 x 12 heads x 1 row, 32 x 256 states of 64 bf16, 62 % valid: 199 us for 1.0 GB, 5.0 TB/s
//   2,048 x 12 x 32 rows, 256 states of 64: 258 us, 4.7 TB/s;  2 x 8 x 4 rows, 100 x 512 states of 128: 65 us, 4.8 TB/s
//   8 x 12 x 48 rows, 100 x 250 states of 64 f16: 135 us, 2.8 TB/s: sixteen products and 64 exponentials a lane for
//   8 KiB, and registers for two waves a SIMD only
template <typename T, int DP, int QB>
__global__ __launch_bounds__(256, 2) void attend_stream_kernel(artread_attend_t A, AttendPlan P, Partials W) {
    constexpr int SLOT = QB * (DP / 2 + 2) * 64;   // floats of a wave's accumulators, maxima and sums
    constexpr int TILES = 4 * 32 * DP * 2, SLOTS = 2 * SLOT * 4;
    __shared__ __attribute__((aligned(1024))) char lds[TILES > SLOTS ? TILES : SLOTS];
    typedef typename Mma<T>::V8 V8;
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = uniform(threadIdx.x >> 6);
    T* tile = (T*)lds + wave * 32 * DP;
    const int dim = (int)A.dim;
    int64_t item = block_id();
    int split = 0, group = 0;
    if (P.walkers == 1) {
        item = item * 4 + wave;
    } else {
        group = (int)(item % P.splits);
        item /= P.splits;
        split = group * 4 + wave;
    }
    if (item >= P.items) return;   // whole workgroups where they have barriers
    const int64_t rb = item % P.row_blocks, bk = item / P.row_blocks;
    const int64_t kh = bk % A.kv_heads, b = bk / A.kv_heads, r0 = rb * 32 * QB + (lane & 31);
    V8 q[QB][DP / 16];
    f32x16 o[QB][DP / 32];
    float m[QB], l[QB];
#pragma unroll
    for (int x = 0; x < QB; ++x) {
        load_q<T, DP>(A, P, (const T*)A.q, A.q_batch, A.q_row, A.q_head, b, kh, r0 + 32 * x, half, P.q_and, P.q_xor, q[x]);
        m[x] = -INFINITY;
        l[x] = 0.0f;
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) o[x][db] = f32x16{};
    }
    const T* kbase = (const T*)A.k + b * A.k_batch + kh * A.k_head + (int64_t)(lane & 31) * A.k_row + 8 * half;
    // V: 8 or 16 lanes per row
    constexpr int CH = DP / 8, VR = 64 / CH, VN = 32 / VR;
    const int vrow = lane / CH, vchunk = lane % CH;
    const T* vbase = (const T*)A.v + b * A.v_batch + kh * A.v_head + (int64_t)vrow * A.v_row + 8 * vchunk;
    V8 kr[DP / 16], vr[VN];
    Walk<32> walk;
    walk.start(A, P, b, split, P.splits * P.walkers);
    auto load = [&]() {
        const uint32_t valid = (uint32_t)walk.mask;
        const T* kp = kbase + walk.p * A.k_passage + walk.j0 * A.k_row;
        const T* vp = vbase + walk.p * A.v_passage + walk.j0 * A.v_row;
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) kr[s] = load8<T>(kp + 16 * s, (valid >> (lane & 31) & 1) && 16 * s + 8 * half < dim);
#pragma unroll
        for (int x = 0; x < VN; ++x) vr[x] = load8<T>(vp + (int64_t)x * VR * A.v_row, (valid >> (vrow + x * VR) & 1) && 8 * vchunk < dim);
    };
    bool more = walk.settle();
    if (more) load();
    while (more) {
        const uint64_t mask = walk.mask;
        f32x16 s[QB][1];
#pragma unroll
        for (int x = 0; x < QB; ++x) s[x][0] = f32x16{};
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
#pragma unroll
            for (int x = 0; x < QB; ++x) s[x][0] = Mma<T>::mul(kr[k], q[x][k], s[x][0]);
#pragma unroll
        for (int x = 0; x < VN; ++x) {
            const int row = vrow + x * VR;
            *(V8*)(tile + row * DP + tile_chunk<DP>(row, vchunk) * 8) = vr[x];
        }
        walk.advance();
        more = walk.settle();
        if (more) load();
#pragma unroll
        for (int x = 0; x < QB; ++x) softmax_tile<T, 1, DP / 32>(s[x], P.c, mask, half, m[x], l[x], o[x]);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the tile is written: LDS keeps a wave's order
        const uint32_t vcol = opaque(lds_offset(tile) + columns_base<DP>(lane));
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            V8 pw[QB];
#pragma unroll
            for (int x = 0; x < QB; ++x) pw[x] = weights8<T>(s[x][0], ks);
#pragma unroll
            for (int db = 0; db < DP / 32; ++db) {
                const V8 vt = lds_columns<T, DP>(vcol, 16 * ks, db);
#pragma unroll
                for (int x = 0; x < QB; ++x) o[x][db] = Mma<T>::mul(vt, pw[x], o[x][db]);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
#pragma unroll
    for (int x = 0; x < QB; ++x) l[x] = both_sum(l[x]);
    if (P.walkers > 1) {
        float* slots = (float*)lds;
#pragma unroll
        for (int step = 2; step; step >>= 1) {
            __syncthreads();   // tiles, and the slots of the step before, are read
            if (wave >= step && wave < 2 * step) {
                float* at = slots + (wave - step) * SLOT + lane;
#pragma unroll
                for (int x = 0; x < QB; ++x) {
                    at[(x * 2) * 64] = m[x];
                    at[(x * 2 + 1) * 64] = l[x];
#pragma unroll
                    for (int i = 0; i < DP / 2; ++i) at[(QB * 2 + x * (DP / 2) + i) * 64] = o[x][i >> 4][i & 15];
                }
            }
            __syncthreads();
            if (wave < step) {
                const float* at = slots + wave * SLOT + lane;
#pragma unroll
                for (int x = 0; x < QB; ++x) {
                    const float m2 = at[(x * 2) * 64], l2 = at[(x * 2 + 1) * 64], m1 = fmaxf(m[x], m2);
                    const float base = m1 == -INFINITY ? 0.0f : m1;   // no key so far: zeros stay zeros
                    const float f = __builtin_amdgcn_exp2f(m[x] - base), f2 = __builtin_amdgcn_exp2f(m2 - base);
                    m[x] = m1;
                    l[x] = l[x] * f + l2 * f2;
#pragma unroll
                    for (int i = 0; i < DP / 2; ++i)
                        o[x][i >> 4][i & 15] = o[x][i >> 4][i & 15] * f + at[(QB * 2 + x * (DP / 2) + i) * 64] * f2;
                }
            }
        }
        if (wave > 0) return;
    }
#pragma unroll
    for (int x = 0; x < QB; ++x) finish_rows<T, DP>(A, P, W, b, kh, r0 + 32 * x, group, half, m[x], l[x], o[x]);
}

// ---- many rows: four waves share the tiles --------------------------------------------------------------
// Workgroups of one (batch entry, key head) sit on one XCD, whose L2 then serves its states.  Its neighbours there are
// of other batch entries, since the heads of one have the same lengths: an XCD of long passages would be waited for
// (8 batch entries of 8 x 512 states, 4 key heads: 302 us against 310).
__device__ __forceinline__ int64_t xcd_item(int64_t id, int64_t items) {
    const int64_t per = (items + 7) / 8;
    return (id >> 3) < per ? (id & 7) * per + (id >> 3) : items;
}

// Brings tiles of KB x 32 states into a ring of LDS: 1 KiB pieces, every NW-th of a tile by one of NW waves.  States
// that are not valid and columns behind dim become zeros: the states are written, the columns cleared once.
template <typename T, int DP, int KB, int NW>
struct TileFetch {
    static constexpr int CH = DP / 8, PR = 64 / CH, PW = 32 * KB / PR / NW;   // chunks per row, rows per piece
    static constexpr int FOLD = DP == 128 ? 3 : 1;    // of a row's place in the order of chunks its piece changes two bits
    static_assert(NW == 1 || NW % 4 == 0, "");
    typedef typename std::conditional<KB == 1, uint32_t, uint64_t>::type Mask;
    int wave;
    __device__ __forceinline__ void start(int w) { wave = w; }
    __device__ __forceinline__ int64_t first(int64_t stride) const { return wave * PR * stride; }
    // src: the wave's first state of the tile (first() from the tile's); mask: which of its states are valid; stride below 2^24
    __device__ __forceinline__ void fetch(const T* src, int64_t stride, Mask mask, int dim, uint32_t tile) const {
        const uint32_t lane = opaque(threadIdx.x & 63), row = lane / CH;   // anew each time: registers are few
        const uint32_t chunk = tile_chunk<DP>(row, lane % CH) ^ ((wave & FOLD) << (DP == 128 ? 0 : 1));
        const uint32_t bytes = (uint32_t)row * (uint32_t)stride * 2;
        uint32_t off[PW];
#pragma unroll
        for (int x = 0; x < PW; ++x) off[x] = bytes + (uint32_t)(chunk ^ ((x * NW & FOLD) << (DP == 128 ? 0 : 1))) * 16;
        tile += (uint32_t)wave * 1024;
        const uint32_t step = (uint32_t)stride * (NW * PR * 2);
        if (whole_tile<KB>(mask)) {   // uniform
            constexpr int N = PW < 4 ? PW : 4;
            if (dim == DP) {
#pragma unroll
                for (int x = 0; x < PW; x += N) dma_pieces<N, NW * 1024>((const char*)src + x * (uint64_t)step, step, off + x, tile + x * (NW * 1024));
                return;
            }
        }
#pragma unroll
        for (int x = 0; x < PW; ++x) {
            const uint32_t piece = x * NW + wave, c = chunk ^ ((x * NW & FOLD) << (DP == 128 ? 0 : 1));
            const uint32_t dst = tile + (uint32_t)x * (NW * 1024);
            if (c * 8 < (uint32_t)dim && (mask >> (piece * PR + row) & 1)) {
                dma16((const char*)src + x * (uint64_t)step, off[x], dst);
            } else if (!whole_tile<KB>(mask)) {
                *(__attribute__((address_space(3))) u32x4*)(uintptr_t)(dst + lane * 16) = u32x4{0, 0, 0, 0};
            }
        }
    }
};

// 128 rows per workgroup, 32 of them a wave's, 64 keys per tile; while a tile is worked on the next one arrives.
// Bound by what a SIMD issues: per tile a wave's 32 products take 1,024 cycles and its other vector instructions about
// as many, a quarter of that the exponentials, and two waves overlap them in part: 46 % of the cycles have a product.
// The two workgroups of a compute unit are what overlaps; measured on 8 x 8 x 512 states of 128 bf16 columns, 75 % valid,
// 4,096 rows a key head (257 us, 800 TFLOP/s; 233 us, 887 back to back): 64 rows a wave 494 us (registers spill), tiles
// of 32 keys in a ring of three 379, three waves a SIMD 385 - each when this took 373; eight waves a workgroup 284
// against 271, the same with three tiles in LDS 305, and two groups of four waves kept half a tile apart by barriers,
// one in the products while the other is in the softmax, 321 against 297.
template <typename T, int DP>
__global__ __launch_bounds__(256, 2) void attend_tile_kernel(artread_attend_t A, AttendPlan P, Partials W) {
    constexpr int KB = 2, TILE = 32 * KB * DP;
    __shared__ __attribute__((aligned(1024))) T ring[4][TILE];   // two tiles of K, two of V
    typedef typename Mma<T>::V8 V8;
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = uniform(threadIdx.x >> 6);
    const int dim = (int)A.dim;
    TileFetch<T, DP, KB, 4> fetcher;
    fetcher.start(wave);
    if (dim < DP) {
        for (int i = threadIdx.x; i < 4 * TILE / 8; i += 256) ((u32x4*)&ring[0][0])[i] = u32x4{0, 0, 0, 0};
        __syncthreads();
    }
    const int64_t total = P.items * P.splits;
    const int64_t w = xcd_item(block_id(), total);
    if (w >= total) return;
    const int64_t rb = w % P.row_blocks, other = w / P.row_blocks;
    const int split = (int)(other % P.splits);
    const int64_t hb = other / P.splits, kh = hb / A.batch, b = hb % A.batch;
    const int64_t r = (rb * 4 + wave) * 32 + (lane & 31);
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
    V8 q[DP / 16];
    f32x16 o[DP / 32];
    float m = -INFINITY, l = 0.0f;
    load_q<T, DP>(A, P, (const T*)A.q, A.q_batch, A.q_row, A.q_head, b, kh, r, half, P.q_and, P.q_xor, q);
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) o[db] = f32x16{};
    int stage = 0;
    while (more) {
        mask = next_mask;
        dma_wait<0>();
        wave_meet();   // everyone's pieces are there, and everyone is done with the tile before
        more = fetch(stage ^ 1);
        const uint32_t krow = opaque(lds_offset(ring[stage]) + rows_base<DP>(lane));
        const uint32_t vcol = opaque(lds_offset(ring[2 + stage]) + columns_base<DP>(lane));
        f32x16 s[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) s[kb] = f32x16{};
        constexpr int NK = KB * DP / 16, NV = 2 * KB * DP / 32, AHEAD = NK < 8 ? NK : 8;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) s[kb] = Mma<T>::mul(lds_rows<T, DP>(krow, kb, k), q[k], s[kb]);
        // the operands of the second product are on their way while the softmax runs
        V8 vt[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) vt[i] = lds_columns<T, DP>(vcol, 16 * (i / (DP / 32)), i % (DP / 32));
        __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);   // LDS reads ahead, then one per product
#pragma unroll
        for (int i = 0; i < NK - AHEAD; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
        __builtin_amdgcn_s_setprio(0);   // the other wave of the SIMD may have its products first
        softmax_tile<T, KB, DP / 32>(s, P.c, mask, half, m, l, o);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int ks = 0; ks < 2 * KB; ++ks) {
            const V8 pw = weights8<T>(s[ks >> 1], ks & 1);
#pragma unroll
            for (int db = 0; db < DP / 32; ++db) o[db] = Mma<T>::mul(vt[ks * (DP / 32) + db], pw, o[db]);
        }
        stage ^= 1;
    }
    finish_rows<T, DP>(A, P, W, b, kh, r, split, half, m, both_sum(l), o);
}
