// block_attn.hip -- softmax attention of every query over the blocks of 64 keys that were picked for it, and its gradient.
//
//   x_ij = scale q_i . k_j  over the live keys j of the picked blocks (causal: j <= n - m + i),
//   p_ij = exp(x_ij) / sum_j exp(x_ij),   o_i = sum_j p_ij v_j,   nothing to see: o_i = 0
//   dv_j = sum_i p_ij do_i,   ds_ij = p_ij (do_i . v_j - do_i . o_i),   dq_i = scale sum_j ds_ij k_j,
//   dk_j = scale sum_i ds_ij q_i
//
// Forward and dq: a workgroup takes 64 rows = 64 / group queries of one key head with all heads of the group (they share
// the picked blocks), forms the UNION of the rows' blocks in LDS with one bit per query, and runs over it once, with the
// running maximum and sum of the softmax.  A block that no row of a wave picked is skipped by that wave; in the others a row
// that did not pick it subtracts infinity from its scores (forward; no instruction more a score) or takes zeros (dq; a select a
// score).  A block's keys and values are read once for 64 rows.  What that costs is the union: queries that are near each other
// pick some of the same blocks -- points in a spatial order, tokens in a sequence, the heads of a group always.  Blocks a query /
// of a wave's 16 rows / of the 64: clouds of 5000 points in the order of a space-filling curve 8 / 16 / 24, rows of a level over
// another's merged cloud 5 / 11 / 20, a causal sequence of 8192 rows 16 / 23 / 30.  Where neighbouring rows are far apart (the
// same clouds shuffled: 8 / 58 / 76 of 79) all is worked on, and a call takes 2.2 times as long.
// dk, dv: a workgroup per block of keys, or, up to 1024 blocks, per part of its queries (ba_dkv_chunk), gathers the rows that
// picked it (a bit matrix, blocks by queries, written by block_pick_bits_kernel) and runs over them densely.  Nothing is added
// up with atomics: results do not depend on the order in which workgroups run.
//
// Matrix instructions: 16x16x32 on the 16-bit types, 16x16x4 on fp32 (eight of them per 32 channels); accumulators, the
// softmax and all sums in fp32.  Scores are formed transposed (keys x rows): a lane then holds 16 scores of ONE row, the
// row's maximum is 15 register operations and two lane exchanges, and the probabilities already sit where the second
// product wants its B operand -- the order of the 32 keys inside an instruction is free as long as both operands agree.
// The transposed operand of that product comes out of the row-major LDS tile through the transposing LDS read.
#include "heads.h"

namespace {

constexpr int BA_BLOCK = TPU3_ATTN_BLOCK;
constexpr int BA_THREADS = 256;
constexpr int BA_ROWS = 64;                 // rows of a workgroup, 16 a wave

struct BaArgs {
    tpu3_heads q, k, v, o, go;              // o, go: backward
    const int32_t *blocks;                  // (b, m, hk, count)
    const int32_t *n_arr, *m_arr;
    void *out, *out2, *dq;                  // forward: o; backward: dk, dv, dq (contiguous)
    void *rest;                             // 16-bit types, contiguous like o: what the rounding of o took (ba_rest_scale), for do . o
    float *lse;                             // (b, hq, m, 2): BaStat of the row
    float *row;                             // (b, hq, m, 2): for dk, dv: BaStat::by of the row there, and do . o
    uint64_t *bits;                         // (b, hk, nb, mt): bit = query of the tile of 64 picked the block
    float *part;                            // split forward: (rows, splits, d + 4); dk / dv in parts: (parts, 2, 64, d)
    int32_t *picks, *first;                 // dk / dv in parts: queries that picked a block; first part of a block, and the end
    uint32_t *unclean;                      // backward: a value that is not finite came out somewhere
    int chunk;                              // queries of a part; 0: a workgroup per block
    int b, m, n, nb, mt, hq, hk, group, d, count, causal, splits, tiles, qt, cap;
    unsigned group_inverse;                 // ceil(2^32 / group): r / group = umulhi(r, it) for r * group < 2^32, group > 1
    float scale, scale2, scale2_rest;       // scale * log2(e) in two terms
};

typedef short ba_s4 __attribute__((ext_vector_type(4)));

// ---- operands ----------------------------------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ hd_f4 ba_mma(const typename hd_vec<T>::v8 &a, const typename hd_vec<T>::v8 &b, hd_f4 c);
template <> __device__ __forceinline__ hd_f4 ba_mma<__bf16>(const hd_bf8 &a, const hd_bf8 &b, hd_f4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
template <> __device__ __forceinline__ hd_f4 ba_mma<_Float16>(const hd_h8 &a, const hd_h8 &b, hd_f4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
template <> __device__ __forceinline__ hd_f4 ba_mma<float>(const hd_f8 &a, const hd_f8 &b, hd_f4 c)
{
#pragma unroll
    for (int i = 0; i < 8; ++i)
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[i], b.v[i], c, 0, 0, 0);
    return c;
}
// The same for scores.  fp32: the 32 products in two sums of 16 of their own, so that only the last addition rounds at the
// score's size: with one chain of D such roundings the output of 96 channels was off by twice the plain form's error (1.3e-6
// against 6e-7; 4e-7 with these).
template <typename T> __device__ __forceinline__ hd_f4 ba_score_mma(const typename hd_vec<T>::v8 &a, const typename hd_vec<T>::v8 &b, hd_f4 c)
{
    if constexpr (sizeof(T) == 2) {
        return ba_mma<T>(a, b, c);
    } else {
        hd_f4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[i], b.v[i], x, 0, 0, 0);
            y = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[4 + i], b.v[4 + i], y, 0, 0, 0);
        }
        return c + (x + y);
    }
}

template <typename T> __device__ __forceinline__ typename hd_vec<T>::v8 ba_zero()
{
    typename hd_vec<T>::v8 z;
    __builtin_memset(&z, 0, sizeof(z));
    return z;
}

// A tile of 64 rows in LDS, unpadded; the 16-byte pieces of a row are permuted by its number (piece ^ f(row), f below) so that
// both kinds of reads hit 64 different banks: 16 lanes that read one piece of 16 consecutive rows, and 32 lanes that read
// 32 bytes of 8 consecutive rows (the transposing read).  256 bytes hold 1, 2 or 4 rows: f runs through the even numbers
// over rows 0 .. 7 (of different 256-byte lines) and through the odd ones over rows 8 .. 15.
template <typename T, int DP> struct BaLds {
    static constexpr int ROWB = DP * (int)sizeof(T), PIECE = 16 / (int)sizeof(T);
    static constexpr size_t TILE = (size_t)BA_ROWS * ROWB;
    static __device__ __forceinline__ int f(int row)
    {
        const int low = ROWB >= 256 ? (row & 7) : ROWB == 128 ? ((row >> 1) & 3) : ((row >> 2) & 1);
        return (low << 1) | ((row >> 3) & 1);
    }
    // place of a row's piece, in elements
    static __device__ __forceinline__ int at(int row, int piece) { return row * DP + ((piece ^ f(row)) * PIECE); }
    // eight channels from 8 * part on
    static __device__ __forceinline__ typename hd_vec<T>::v8 row8(const T *tile, int row, int part)
    {
        if constexpr (sizeof(T) == 2) {
            return *(const typename hd_vec<T>::v8 *)(tile + at(row, part));
        } else {
            hd_f8 r;
            *(hd_f4 *)(r.v) = *(const hd_f4 *)(tile + at(row, 2 * part));
            *(hd_f4 *)(r.v + 4) = *(const hd_f4 *)(tile + at(row, 2 * part + 1));
            return r;
        }
    }
    static __device__ __forceinline__ void put8(T *tile, int row, int part, const typename hd_vec<T>::v8 &x)
    {
        if constexpr (sizeof(T) == 2) {
            *(typename hd_vec<T>::v8 *)(tile + at(row, part)) = x;
        } else {
            *(hd_f4 *)(tile + at(row, 2 * part)) = hd_f4{x.v[0], x.v[1], x.v[2], x.v[3]};
            *(hd_f4 *)(tile + at(row, 2 * part + 1)) = hd_f4{x.v[4], x.v[5], x.v[6], x.v[7]};
        }
    }
    // A operand, transposed: lane (l15, g) gets channel 16 * c + l15 of the rows r0 + g*4 + {0..3} and r0 + 16 + g*4 + {0..3}
    static __device__ __forceinline__ typename hd_vec<T>::v8 column(const T *tile, int r0, int c)
    {
        const int lane = threadIdx.x & 63, g = lane >> 4, l15 = lane & 15;
        typename hd_vec<T>::v8 o;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                o.v[i] = tile[at(r0 + g * 4 + i, c * 4 + (l15 >> 2)) + (l15 & 3)];
                o.v[4 + i] = tile[at(r0 + 16 + g * 4 + i, c * 4 + (l15 >> 2)) + (l15 & 3)];
            }
        } else {
            // 16 lanes read a 4 x 16 piece (8 bytes a lane) and receive its columns
            typedef __attribute__((address_space(3))) ba_s4 lds_s4;
            const T *p = tile + at(r0 + g * 4 + (l15 >> 2), c * 2 + ((l15 >> 1) & 1)) + (l15 & 1) * 4;
            union {
                ba_s4 s[2];
                typename hd_vec<T>::v8 v;
            } u;
            u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(p));
            u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(p + 16 * DP));
            o = u.v;
        }
        return o;
    }
};

template <typename T> __device__ __forceinline__ typename hd_vec<T>::v8 ba_pack(const hd_f4 &a, const hd_f4 &b)
{
    typename hd_vec<T>::v8 f;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            f.v[i] = a[i], f.v[4 + i] = b[i];
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            f[i] = (T)a[i], f[4 + i] = (T)b[i];
    }
    return f;
}

// what rounding a and b to f took
template <typename T> __device__ __forceinline__ typename hd_vec<T>::v8 ba_rest(const hd_f4 &a, const hd_f4 &b, const typename hd_vec<T>::v8 &f)
{
    hd_f4 r0, r1;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        r0[i] = a[i] - (float)f[i], r1[i] = b[i] - (float)f[4 + i];
    return ba_pack<T>(r0, r1);
}

template <typename T> __device__ __forceinline__ void ba_store4(T *p, const hd_f4 &x)
{
    typename hd_vec<T>::v4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        y[i] = (T)x[i];
    *(typename hd_vec<T>::v4 *)p = y;
}

// What the rounding of o took, as it is stored: fp16 times 2^11 (at most 2^15, and a step of 2^-35 where o itself is below the
// normal numbers).
template <typename T> __device__ __forceinline__ constexpr float ba_rest_scale() { return __is_same(T, _Float16) ? 2048.f : 1.f; }

// the same, and what the rounding took
template <typename T> __device__ __forceinline__ void ba_store_rest(T *p, T *rest, bool want, int at, const hd_f4 &x)
{
    ba_store4<T>(p + at, x);
    if (sizeof(T) == 2 && want) {
        hd_f4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            r[i] = (x[i] - (float)(T)x[i]) * ba_rest_scale<T>();
        ba_store4<T>(rest + at, r);
    }
}

// maximum / sum over the four lane groups that hold a column (lanes l, l+16, l+32, l+48): swapping a register with itself
// between halves (rows) of the wave gives both sides' values, without a trip through LDS
__device__ __forceinline__ float ba_col_max(float v)
{
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float ba_col_sum(float v)
{
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// ---- staging of a 64-row tile ------------------------------------------------------------------------------------------
template <typename T, int DP> struct BaStage {
    typedef BaLds<T, DP> L;
    static constexpr int PARTS = DP / 8, PER = BA_ROWS * PARTS / BA_THREADS;                // eight-channel parts of a thread
    typename hd_vec<T>::v8 r[PER];
    static constexpr int STEP = BA_THREADS / PARTS;
    static __device__ __forceinline__ int row(int i) { return (int)threadIdx.x / PARTS + i * STEP; }
    static __device__ __forceinline__ int part(int) { return (int)threadIdx.x % PARTS; }
    // Rows [row0, row0 + 64) of one head.  Rows from `end` on are the last one's copies and channels from d on channel 0's:
    // real numbers, whose scores are masked or meet zeros.  `lane`: this thread's place in the head (BaStage::lane).
    static __device__ __forceinline__ const T *lane(const T *base, int d) { return base + (part(0) * 8 < d ? part(0) * 8 : 0); }
    __device__ __forceinline__ void load(const T *lane, int64_t stride, int row0, int end)
    {
#pragma unroll
        for (int i = 0; i < PER; ++i)
            r[i] = *(const typename hd_vec<T>::v8 *)(lane + min(row0 + row(i), end - 1) * stride);
    }
    // the tile with what is not finite as zero; `odd` collects the rows that hold such a value
    __device__ __forceinline__ void store_finite(T *tile, unsigned long long *odd) const
    {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            typename hd_vec<T>::v8 x = r[i];
            bool any = false;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const bool fin = fabsf((float)r[i][c]) <= 3.4028235e38f;
                any |= !fin;
                if constexpr (sizeof(T) == 4)
                    x.v[c] = fin ? x.v[c] : 0.f;
                else
                    x[c] = fin ? x[c] : (T)0.f;
            }
            L::put8(tile, row(i), part(i), x);
            if (any)
                atomicOr(odd, 1ull << row(i));
        }
    }
    __device__ __forceinline__ void store(T *tile) const
    {
#pragma unroll
        for (int i = 0; i < PER; ++i)
            L::put8(tile, row(i), part(i), r[i]);
    }
};

// How a kernel is laid out over registers and LDS; w: waves a SIMD that the register allocation aims at.  More waves hide
// more of the chain scores -> maximum -> exponentials -> product, until the operands no longer fit: measured on clouds
// of 5000 points (64 channels) and a sequence of 8192 (128), us with 2 / 3 / 4 waves: forward - / 144 / 129 and
// 310 / 279 / -, dq - / 94 / 99 and 341 / 520 / -, dk and dv - / 63 / 92 and 346 / 900 / - (all before their
// second terms); fp32 of 24 channels, forward, - / 59 / 49.  A wave has 16 rows (keys):
// with 32, every operand read from LDS feeds two matrix instructions, but half as many waves are there (188 for 146).
// together: 16-row tiles whose row operands are read in one go; columns: 16-channel columns read in one go.
template <typename T, int DP> struct BaFwd {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int w = F32 ? (DP == 128 ? 1 : DP == 64 ? 2 : 4) : DP == 128 ? 3 : 4;
    static constexpr int together = F32 ? (DP == 32 ? 4 : DP == 64 ? 2 : 1) : DP == 128 ? 1 : 2;
    static constexpr int columns = DP / 16 < 4 ? DP / 16 : 4;
};
template <typename T, int DP> struct BaBwd {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int w = F32 ? (DP == 128 ? 1 : DP == 64 ? 2 : 3) : DP == 128 ? 2 : 3;
    static constexpr int together = F32 ? (DP == 32 ? 4 : DP == 64 ? 2 : 1) : DP == 128 ? 2 : 4;
    static constexpr int columns = DP / 16;
    static constexpr int kw = F32 ? (DP == 128 ? 1 : 2) : DP == 128 ? 2 : 3;
};
// LDS reads above stay above: the compiler otherwise sinks each to its matrix instruction and waits for it there
__device__ __forceinline__ void ba_issue() { __builtin_amdgcn_sched_barrier(0); }

struct BaTile {                             // which rows a workgroup has
    int b, h, i0, live, lm, z;              // sequence, key head, first query, live keys and queries, split
};
__device__ __forceinline__ BaTile ba_tile(const BaArgs &a, int64_t id)
{
    BaTile t;
    t.z = (int)(id % a.splits);
    id /= a.splits;
    const int tile = (int)(id % a.tiles);
    const int bh = (int)(id / a.tiles);
    t.h = bh % a.hk;
    t.b = bh / a.hk;
    t.i0 = tile * a.qt;
    t.live = a.n_arr ? min(max(a.n_arr[t.b], 0), a.n) : a.n;
    t.lm = a.m_arr ? min(max(a.m_arr[t.b], 0), a.m) : a.m;
    return t;
}
// workgroups are dealt to the eight XCDs in turn: give each XCD a contiguous range of ids, so that the tiles of a head,
// which read the same keys, share an L2
__device__ __forceinline__ int64_t ba_xcd(int64_t id, int64_t all)
{
    const int64_t per = all / 8, cut = per * 8;
    return id < cut ? (id & 7) * per + (id >> 3) : id;
}

// keys that query i may see end here
__device__ __forceinline__ int ba_limit(const BaArgs &a, int live, int lm, int i)
{
    if (i >= lm)
        return 0;
    return a.causal ? max(0, live - lm + i + 1) : live;
}

// The union of the blocks of the tile's queries, ascending, with the queries that picked each: list[u], mask[u], u < the
// return value.  An index outside the live blocks, or behind what the query may see, is nobody's; one that a query names
// twice counts once.
__device__ int ba_union(const BaArgs &a, const BaTile &t, uint32_t *list, uint64_t *mask, uint32_t *words, uint32_t *before)
{
    __shared__ uint32_t wave_total[4];
    const int nw = (a.nb + 31) / 32, entries = a.qt * a.count;
    for (int w = threadIdx.x; w < nw; w += BA_THREADS)
        words[w] = 0;
    __syncthreads();
    const int32_t *idx = a.blocks + (((int64_t)t.b * a.m + t.i0) * a.hk + t.h) * a.count;
    auto entry = [&](int e, int &q) {
        q = e / a.count;
        const int i = t.i0 + q;
        if (i >= t.lm)
            return -1;
        const int blk = idx[(int64_t)q * a.hk * a.count + (e - q * a.count)];
        return blk >= 0 && blk < a.nb && blk * BA_BLOCK < ba_limit(a, t.live, t.lm, i) ? blk : -1;
    };
    constexpr int KEPT = 4;                 // of a thread's entries, in registers between the two passes
    int kept[KEPT];
#pragma unroll
    for (int x = 0; x < KEPT; ++x) {
        const int e = x * BA_THREADS + threadIdx.x;
        int q;
        kept[x] = e < entries ? entry(e, q) : -1;
    }
    auto all_entries = [&](auto &&f) __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < KEPT; ++x)
            if (kept[x] >= 0)
                f(kept[x], (x * BA_THREADS + (int)threadIdx.x) / a.count);
        for (int e = KEPT * BA_THREADS + threadIdx.x; e < entries; e += BA_THREADS) {
            int q;
            const int blk = entry(e, q);
            if (blk >= 0)
                f(blk, q);
        }
    };
    all_entries([&](int blk, int) { atomicOr(words + (blk >> 5), 1u << (blk & 31)); });
    __syncthreads();
    const int per = (nw + BA_THREADS - 1) / BA_THREADS, w0 = min(nw, (int)threadIdx.x * per), w1 = min(nw, w0 + per);
    uint32_t mine = 0;
    for (int w = w0; w < w1; ++w)
        mine += __popc(words[w]);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t inc = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t v = __shfl_up(inc, o, 64);
        inc += lane >= o ? v : 0u;
    }
    if (lane == 63)
        wave_total[wave] = inc;
    __syncthreads();
    uint32_t at = inc - mine, total = 0;
    for (int w = 0; w < BA_THREADS / 64; ++w) {
        at += w < wave ? wave_total[w] : 0u;
        total += wave_total[w];
    }
    for (int w = w0; w < w1; ++w) {
        before[w] = at;
        at += __popc(words[w]);
    }
    for (uint32_t u = threadIdx.x; u < total; u += BA_THREADS)
        mask[u] = 0;
    __syncthreads();
    auto slot = [&](int blk) { return before[blk >> 5] + __popc(words[blk >> 5] & ((1u << (blk & 31)) - 1)); };
    all_entries([&](int blk, int q) {
        const uint32_t u = slot(blk);
        list[u] = (uint32_t)blk;            // (all that name the block write the same)
        atomicOr((unsigned long long *)(mask + u), 1ull << q);
    });
    __syncthreads();
    return (int)total;
}

// the rows of this lane's column as B operands: channels kk*32 + g*8 .. +8 of row l15
template <typename T, int DP>
__device__ __forceinline__ void ba_row_operand(const T *p, bool live, int d, typename hd_vec<T>::v8 *f)
{
    const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int kk = 0; kk < DP / 32; ++kk) {
        const int c = kk * 32 + g * 8;
        f[kk] = live && c < d ? *(const typename hd_vec<T>::v8 *)(p + c) : ba_zero<T>();
    }
}

// ---- forward -----------------------------------------------------------------------------------------------------------
// This lane's row (column of the transposed scores) in the forward and the dq kernel.
struct BaRow {
    int ql, i, head, limit;
    bool mine, there;
    __device__ __forceinline__ BaRow(const BaArgs &a, const BaTile &t)
    {
        const int row = (threadIdx.x >> 6) * 16 + (threadIdx.x & 15);
        ql = row / a.group;
        i = t.i0 + ql;
        head = t.h * a.group + (row - ql * a.group);
        there = ql < a.qt && i < a.m;
        mine = there && i < t.lm;
        limit = mine ? ba_limit(a, t.live, t.lm, i) : 0;
    }
    template <typename T> __device__ __forceinline__ const T *at(const tpu3_heads &x, int b) const
    {
        return (const T *)x.data + b * x.sb + (int64_t)i * x.sr + (int64_t)head * x.sh;
    }
    __device__ __forceinline__ int64_t flat(const BaArgs &a, int b) const { return ((int64_t)b * a.hq + head) * a.m + i; }
    __device__ __forceinline__ int64_t out(const BaArgs &a, int b) const { return (((int64_t)b * a.m + i) * a.hq + head) * a.d; }
};

// scores (keys x rows) of the tile: s[x] = 16 keys x 16 rows
template <typename T, int DP, int TG>
__device__ __forceinline__ void ba_scores(const T *tile, const typename hd_vec<T>::v8 *f, hd_f4 *s)
{
    typedef BaLds<T, DP> L;
    const int lane = threadIdx.x & 63, l15 = lane & 15, g = lane >> 4;
#pragma unroll
    for (int x0 = 0; x0 < 4; x0 += TG) {
        typename hd_vec<T>::v8 kf[TG][DP / 32];
#pragma unroll
        for (int x = 0; x < TG; ++x)
#pragma unroll
            for (int kk = 0; kk < DP / 32; ++kk)
                kf[x][kk] = L::row8(tile, (x0 + x) * 16 + l15, kk * 4 + g);
        ba_issue();
#pragma unroll
        for (int x = 0; x < TG; ++x)
            s[x0 + x] = hd_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < DP / 32; ++kk)
#pragma unroll
            for (int x = 0; x < TG; ++x)
                s[x0 + x] = ba_score_mma<T>(kf[x][kk], f[kk], s[x0 + x]);
    }
}
// acc[d] += (tile's columns) (f[0] for its first 32 rows, f[1] for the others): a group of columns is read while the matrix
// instructions of the one before run.  start() reads the first group; before(j) runs ahead of half j's matrix instructions.
template <typename T, int DP, int VG> struct BaColumns {
    static constexpr int STEPS = 2 * (DP / 16) / VG;
    typename hd_vec<T>::v8 c[2][VG];
    __device__ __forceinline__ void read(const T *tile, int step)
    {
#pragma unroll
        for (int i = 0; i < VG; ++i)
            c[step & 1][i] = BaLds<T, DP>::column(tile, step >= STEPS / 2 ? 32 : 0, (step % (STEPS / 2)) * VG + i);
    }
    __device__ __forceinline__ void start(const T *tile)
    {
        read(tile, 0);
        ba_issue();
    }
    // before(j): the operand f[j]; REST adds a second term of it, after(j)
    template <bool REST, typename F, typename G>
    __device__ __forceinline__ void run(const T *tile, hd_f4 *acc, F &&before, G &&after)
    {
        typename hd_vec<T>::v8 f, f2;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            if (s % (STEPS / 2) == 0)
                f = before(s / (STEPS / 2));
            if constexpr (REST)
                if (s % (STEPS / 2) == 0)
                    f2 = after(s / (STEPS / 2), f);
            if (s + 1 < STEPS) {
                read(tile, s + 1);
                ba_issue();
            }
#pragma unroll
            for (int i = 0; i < VG; ++i) {
                hd_f4 &x = acc[(s % (STEPS / 2)) * VG + i];
                x = ba_mma<T>(c[s & 1][i], f, x);
            }
            if constexpr (REST) {
#pragma unroll
                for (int i = 0; i < VG; ++i) {
                    hd_f4 &x = acc[(s % (STEPS / 2)) * VG + i];
                    x = ba_mma<T>(c[s & 1][i], f2, x);
                }
            }
        }
    }
};
// 2^(scaled d + shift), d = a score less its row's largest.  The difference comes first: near the largest score, where the weight
// is, it is exact however large the scores are (scaled ones of 2^31 and more had no or infinite weight when the difference was of
// their rounded products, and the gradients' probabilities were off by half a step of the largest score).  fp32 takes the
// scale's second term too: its rounding moves a difference of 20 by as much as all of an fp32 result's other roundings.
template <typename T> __device__ __forceinline__ float ba_power(const BaArgs &a, float d, float shift)
{
    float e = __builtin_fmaf(d, a.scale2, shift);
    if constexpr (sizeof(T) == 4)
        e = __builtin_fmaf(d, a.scale2_rest, e);
    return __builtin_amdgcn_exp2f(e);
}
// The forward's weights are 2^shift at the most.  2^-13: a row adds up at most 64 blocks of 64 keys, so that no sum of weighted
// values leaves the range that the values are in (at 1, 20 blocks of values of 3e38 came out infinite).  fp16, whose sums are
// far from fp32's ends: 2^15, for the terms' sake (2^-14 is its last normal number).
template <typename T> __device__ __forceinline__ constexpr float ba_weight_shift() { return __is_same(T, _Float16) ? 15.f : -13.f; }

// What the backward pass takes of a row's softmax: the largest score, and of the sum minus its log2, or in fp32, where the rounding
// of a log2 of up to 12 is as much as all other roundings together (dq of 24 channels off by 1.9 times the plain form's), its
// reciprocal.  A row without weights (nothing seen, or scores of -infinity only; its output is 0) has p = 0 whatever its scores
// are; a sum that is not a number: no more is p.
struct BaStat {
    float top, by;
};
template <typename T> __device__ __forceinline__ float ba_probability(const BaArgs &a, float score, float top, float by)
{
    return sizeof(T) == 4 ? ba_power<T>(a, score - top, 0.f) * by : ba_power<T>(a, score - top, by);
}
template <typename T> __device__ __forceinline__ void ba_put_row(const BaArgs &a, int64_t row, float top, float sum)
{
    constexpr bool F32 = sizeof(T) == 4;
    a.lse[2 * row] = sum == 0.f ? (F32 ? INFINITY : 0.f) : top;
    a.lse[2 * row + 1] = F32 ? (sum == 0.f ? 0.f : 0x1p-13f / sum) : sum == 0.f ? -INFINITY : ba_weight_shift<T>() - log2f(sum);
    static_assert(!F32 || ba_weight_shift<T>() == -13.f, "");
}
__device__ __forceinline__ bool ba_finite(float x) { return fabsf(x) <= 3.4028235e38f; }

// one block of keys: Ks, with Vs behind it, in LDS; k0 = its first key; bit = this lane's row picked it
template <typename T, int DP, bool CAREFUL>
__device__ __forceinline__ void ba_fwd_block(const BaArgs &a, const BaRow &R, const typename hd_vec<T>::v8 *qf, const T *Ks, const T *V,
                                             int k0, bool bit, const unsigned long long *odd, hd_f4 *acc, hd_f4 &sums, float &top)
{
    typedef typename hd_vec<T>::v8 V8;
    const T *Vs = Ks + BA_ROWS * DP;
    const int lane = threadIdx.x & 63, l15 = lane & 15, g = lane >> 4;
    if (!__any(bit))
        return;                         // (wave-uniform)
    hd_f4 s[4];
    ba_scores<T, DP, BaFwd<T, DP>::together>(Ks, qf, s);
    BaColumns<T, DP, BaFwd<T, DP>::columns> vc;
    vc.start(Vs);
    if (__any(bit && k0 + BA_BLOCK > R.limit)) {
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                s[x][r] = k0 + x * 16 + g * 4 + r < R.limit ? s[x][r] : -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            mx = fmaxf(mx, s[x][r]);
    mx = ba_col_max(mx);
    const float next = bit ? fmaxf(top, mx) : top;
    const float base = next == -INFINITY ? 0.f : next;
    const float keep = ba_power<T>(a, top - base, 0.f);             // top = -inf: 0
    top = next;
    if (__any(keep != 1.f)) {
        sums *= keep;
#pragma unroll
        for (int d = 0; d < DP / 16; ++d)
            acc[d] *= keep;
    }
    // a row that did not pick the block: 2^(x - inf) = 0 (a score that is not finite is left to the careful pass)
    const float off = bit ? base : INFINITY;
    auto weight = [&](int x) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            s[x][r] = ba_power<T>(a, s[x][r] - off, ba_weight_shift<T>());
            if (CAREFUL)
                s[x][r] = bit ? s[x][r] : 0.f;
        }
    };
    // the denominator: this lane's share by additions, of the probabilities as they are; the product takes them in two terms of a
    // 16-bit type (in one, the output was off by 1.25 times what its last rounding takes: bf16 0.0021 for 0.0017)
    vc.template run<sizeof(T) == 2>(
        Vs, acc,
        [&](int j) __attribute__((always_inline)) {
            weight(2 * j), weight(2 * j + 1);
            sums += s[2 * j] + s[2 * j + 1];
            return ba_pack<T>(s[2 * j], s[2 * j + 1]);
        },
        [&](int j, const V8 &f) __attribute__((always_inline)) { return ba_rest<T>(s[2 * j], s[2 * j + 1], f); });
    if constexpr (CAREFUL) {
        for (unsigned long long left = *odd; left; left &= left - 1) {
            const int kk = __ffsll(left) - 1;                   // the key's place in the block: score register and lane group
            float p = 0.f;
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    p = (kk >> 4) == x && (kk & 3) == r ? s[x][r] : p;
            p = __shfl(p, ((kk >> 2) & 3) * 16 + l15, 64);
            const bool sees = bit && k0 + kk < R.limit;
#pragma unroll
            for (int d = 0; d < DP / 16; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int ch = d * 16 + g * 4 + r;
                    const float val = sees && ch < a.d ? (float)V[(int64_t)(k0 + kk) * a.v.sr + ch] : 0.f;
                    if (!ba_finite(val))
                        acc[d][r] = __builtin_fmaf(p, val, acc[d][r]);
                }
        }
    }
}

// A value that is not finite, times the probability 0 of a row that does not see it, is not 0: in the matrix product it would
// reach every row of the wave.  A workgroup that ends with such an output runs its blocks a second time, carefully: these
// values stay out of the matrix product and are added to the rows that see them one by one.
template <typename T, int DP, bool CAREFUL>
__device__ __forceinline__ void ba_fwd_pass(const BaArgs &a, const BaTile &t, const BaRow &R, const typename hd_vec<T>::v8 *qf, char *smem,
                                            const uint64_t *mask, const uint32_t *list, int count, unsigned long long *odd,
                                            hd_f4 *acc, hd_f4 &sums, float &top)
{
    typedef BaLds<T, DP> L;
    typedef BaStage<T, DP> S;
    const T *K = (const T *)a.k.data + t.b * a.k.sb + t.h * a.k.sh, *V = (const T *)a.v.data + t.b * a.v.sb + t.h * a.v.sh;
    const T *Kl = S::lane(K, a.d), *Vl = S::lane(V, a.d);
#pragma unroll
    for (int d = 0; d < DP / 16; ++d)
        acc[d] = hd_f4{0.f, 0.f, 0.f, 0.f};
    top = -INFINITY, sums = hd_f4{0.f, 0.f, 0.f, 0.f};
    // (a second tile buffer and one barrier less a block made no difference: 142 for 144 us)
    S kr, vr;
    auto fetch = [&](int u) __attribute__((always_inline)) {
        if (u < count) {
            const int r0 = (int)list[u] * BA_BLOCK;
            kr.load(Kl, a.k.sr, r0, t.live);
            vr.load(Vl, a.v.sr, r0, t.live);
        }
    };
    T *k = (T *)smem, *v = (T *)(smem + L::TILE);
    auto put = [&]() __attribute__((always_inline)) {
        kr.store(k);
        if constexpr (CAREFUL) {
            if (threadIdx.x == 0)
                *odd = 0;
            __syncthreads();
            vr.store_finite(v, odd);
        } else {
            vr.store(v);
        }
    };
    fetch(t.z);
    for (int u = t.z; u < count; u += a.splits) {
        __syncthreads();
        put();
        __syncthreads();
        fetch(u + a.splits);
        ba_fwd_block<T, DP, CAREFUL>(a, R, qf, k, V, (int)list[u] * BA_BLOCK, R.mine && ((mask[u] >> R.ql) & 1), odd, acc, sums, top);
    }
}

template <typename T, int DP>
__global__ __launch_bounds__(BA_THREADS, (BaFwd<T, DP>::w)) void block_attn_fwd_kernel(BaArgs a, int64_t all)
{
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ unsigned long long odd;   // careful pass: rows of a tile that hold a value that is not finite
    typedef BaLds<T, DP> L;
    uint64_t *mask = (uint64_t *)(smem + 2 * L::TILE);
    uint32_t *list = (uint32_t *)(mask + a.cap), *words = list + a.cap, *before = words + (a.nb + 31) / 32;

    const int64_t id = ba_xcd(blockIdx.x, all);
    const BaTile t = ba_tile(a, id);
    const int g = (threadIdx.x & 63) >> 4;
    const BaRow R(a, t);
    typename hd_vec<T>::v8 qf[DP / 32];
    ba_row_operand<T, DP>(R.at<T>(a.q, t.b), R.mine, a.d, qf);
    const int count = ba_union(a, t, list, mask, words, before);

    hd_f4 acc[DP / 16], sums;               // sums: running sum of the row
    float top;                              // running maximum of the row's scores
    ba_fwd_pass<T, DP, false>(a, t, R, qf, smem, mask, list, count, &odd, acc, sums, top);
    bool finite = ba_finite(sums[0] + sums[1] + sums[2] + sums[3]);
#pragma unroll
    for (int d = 0; d < DP / 16; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            finite &= ba_finite(acc[d][r]);
    if (__syncthreads_or(!finite))
        ba_fwd_pass<T, DP, true>(a, t, R, qf, smem, mask, list, count, &odd, acc, sums, top);
    const float sum = ba_col_sum(sums[0] + sums[1] + sums[2] + sums[3]);
    if (!R.there)
        return;
    if (a.splits > 1) {
        float *P = a.part + (R.flat(a, t.b) * a.splits + t.z) * (DP + 4);
#pragma unroll
        for (int d = 0; d < DP / 16; ++d)
            *(hd_f4 *)(P + d * 16 + g * 4) = acc[d];
        if (g == 0)
            P[DP] = top, P[DP + 1] = sum;
        return;
    }
    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : NAN;
    const int64_t at = R.out(a, t.b);
#pragma unroll
    for (int d = 0; d < DP / 16; ++d)
        if (d * 16 + g * 4 < a.d)
            ba_store_rest<T>((T *)a.out + at, (T *)a.rest + at, a.rest != nullptr, d * 16 + g * 4, acc[d] * inv);
    if (a.lse && g == 0)
        ba_put_row<T>(a, R.flat(a, t.b), top, sum);
}

// Joins the splits of a row, RL lanes a row (16, or a wave for more splits): a lane per split forms the splits' factors, then a
// lane per DP / RL channels adds the splits up, eight loads at a time.
template <typename T, int DP, int RL>
__global__ __launch_bounds__(BA_THREADS) void block_attn_join_kernel(BaArgs a, int64_t rows)
{
    constexpr int W = DP / RL > 0 ? DP / RL : 1;
    __shared__ float factor[BA_THREADS];
    const int lane = threadIdx.x % RL, first = threadIdx.x - lane;
    const int64_t row = (int64_t)blockIdx.x * (BA_THREADS / RL) + threadIdx.x / RL;
    if (row >= rows)
        return;
    const float *P = a.part + row * a.splits * (DP + 4);
    const float mine = lane < a.splits ? P[lane * (DP + 4) + DP] : -INFINITY, part = lane < a.splits ? P[lane * (DP + 4) + DP + 1] : 0.f;
    float top = mine;
#pragma unroll
    for (int o = RL / 2; o > 0; o >>= 1)
        top = fmaxf(top, __shfl_xor(top, o, 64));
    const float base = top == -INFINITY ? 0.f : top, f = ba_power<T>(a, mine - base, 0.f);
    float sum = part * f;
#pragma unroll
    for (int o = RL / 2; o > 0; o >>= 1)
        sum += __shfl_xor(sum, o, 64);
    factor[threadIdx.x] = f;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : NAN;
    const int64_t i = row % a.m, bh = row / a.m, h = bh % a.hq, b = bh / a.hq;
    const int64_t at = ((b * a.m + i) * a.hq + h) * a.d;
    if (a.lse && lane == 0)
        ba_put_row<T>(a, row, top, sum);
    if (lane * W >= a.d)
        return;
    float y[W] = {};
#pragma unroll 8
    for (int z = 0; z < a.splits; ++z)
#pragma unroll
        for (int c = 0; c < W; ++c)
            y[c] = __builtin_fmaf(P[z * (DP + 4) + lane * W + c], factor[first + z], y[c]);
#pragma unroll
    for (int c = 0; c < W; ++c) {
        const T v = (T)(y[c] * inv);
        ((T *)a.out)[at + lane * W + c] = v;
        if (a.rest)
            ((T *)a.rest)[at + lane * W + c] = (T)((y[c] * inv - (float)v) * ba_rest_scale<T>());
    }
}

// ---- backward: dq, and the rows' do . o ----------------------------------------------------------------------------------
// fp16: two terms of the type hold a number to 2^-22 of it only from 2^-3 on, and to 2^-25 at best, and ds may be of any size.  Its
// row (in dk: its key) is therefore taken times a power of two, `up`, that starts high and is lowered, with what has been added
// up, whenever the largest |ds| so far would pass 2^15: to where that is 2^10 .. 2^11, so that it is seldom lowered twice.  (A power
// from the largest |do| alone left ds of small values or small probabilities below fp16's normal numbers: values of 1e-3, |do| of
// 256: errors of dq and dk 9 times the last rounding's.)  Rows (keys) do not share powers: none loses digits to another's ds.
constexpr float BA_UP = 1.2676506002282294e30f;                 // 2^100
constexpr float BA_P_SHIFT = 15.f;                              // fp16, dk and dv: probabilities times 2^15

// brings x to [2^10, 2^11), within 2^-100 .. 2^100
__device__ __forceinline__ float ba_pow2_to_1024(float x)
{
    const int e = (int)((__float_as_uint(x) >> 23) & 255u);
    return __uint_as_float((uint32_t)min(max(264 - e, 27), 227) << 23);
}
// lowers up, and sums with it, where big * up would pass 2^15; big: the lane's column's largest |ds|
template <int N> __device__ __forceinline__ void ba_lower(float big, float &up, hd_f4 (&sums)[N])
{
    const bool passes = big * up > 32768.f;
    if (!__any(passes))
        return;
    const float next = passes ? ba_pow2_to_1024(big) : up, keep = next / up;
    up = next;
#pragma unroll
    for (int d = 0; d < N; ++d)
        sums[d] *= keep;
}

template <typename T, int DP>
__device__ __forceinline__ void ba_dq_block(const BaArgs &a, const BaRow &R, const typename hd_vec<T>::v8 *qf, const typename hd_vec<T>::v8 *gf,
                                            const BaStat &stat, float delta, float &up, const T *Ks, int k0, bool bit, hd_f4 (&acc)[DP / 16])
{
    typedef typename hd_vec<T>::v8 V8;
    constexpr bool HALF = __is_same(T, _Float16);
    const T *Vs = Ks + BA_ROWS * DP;
    const int g = (threadIdx.x & 63) >> 4;
    if (!__any(bit))
        return;                             // (wave-uniform)
    hd_f4 s[4], dp[4];
    ba_scores<T, DP, BaBwd<T, DP>::together>(Ks, qf, s);
    ba_scores<T, DP, BaBwd<T, DP>::together>(Vs, gf, dp);
    BaColumns<T, DP, BaBwd<T, DP>::columns> kc;
    kc.start(Ks);
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            s[x][r] = ba_probability<T>(a, s[x][r], stat.top, stat.by) * (dp[x][r] - delta);
    if (__any(bit && k0 + BA_BLOCK > R.limit)) {
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                s[x][r] = k0 + x * 16 + g * 4 + r < R.limit ? s[x][r] : 0.f;
    }
    if (!__all(bit)) {
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                s[x][r] = bit ? s[x][r] : 0.f;
    }
    if constexpr (HALF) {
        float big = 0.f;
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                big = fmaxf(big, fabsf(s[x][r]));
        ba_lower(ba_col_max(big), up, acc);
#pragma unroll
        for (int x = 0; x < 4; ++x)
            s[x] *= up;
    }
    // A row's ds add up to nothing, so its dq is what is left of large terms: ds enters in two terms of the 16-bit type (one
    // alone: an error of twice the result's own rounding)
    kc.template run<sizeof(T) == 2>(
        Ks, acc, [&](int j) __attribute__((always_inline)) { return ba_pack<T>(s[2 * j], s[2 * j + 1]); },
        [&](int j, const V8 &f) __attribute__((always_inline)) { return ba_rest<T>(s[2 * j], s[2 * j + 1], f); });
}

// As in the forward kernel, CAREFUL is for tiles in which a key that is not finite may have reached rows that do not see it;
// those that do are not numbers (poison).
template <typename T, int DP, bool CAREFUL>
__device__ __forceinline__ void ba_dq_pass(const BaArgs &a, const BaTile &t, const BaRow &R, const typename hd_vec<T>::v8 *qf,
                                           const typename hd_vec<T>::v8 *gf, const BaStat &stat, float delta, float &up, char *smem,
                                           const uint64_t *mask, const uint32_t *list, int count, unsigned long long *odd,
                                           hd_f4 (&acc)[DP / 16], bool &poison)
{
    typedef BaLds<T, DP> L;
    typedef BaStage<T, DP> S;
    up = BA_UP;
    const T *Kl = S::lane((const T *)a.k.data + t.b * a.k.sb + t.h * a.k.sh, a.d);
    const T *Vl = S::lane((const T *)a.v.data + t.b * a.v.sb + t.h * a.v.sh, a.d);
#pragma unroll
    for (int d = 0; d < DP / 16; ++d)
        acc[d] = hd_f4{0.f, 0.f, 0.f, 0.f};
    S kr, vr;
    auto fetch = [&](int u) __attribute__((always_inline)) {
        if (u < count) {
            const int r0 = (int)list[u] * BA_BLOCK;
            kr.load(Kl, a.k.sr, r0, t.live);
            vr.load(Vl, a.v.sr, r0, t.live);
        }
    };
    T *k = (T *)smem, *v = (T *)(smem + L::TILE);
    auto put = [&]() __attribute__((always_inline)) {
        vr.store(v);
        if constexpr (CAREFUL) {
            if (threadIdx.x == 0)
                *odd = 0;
            __syncthreads();
            kr.store_finite(k, odd);
        } else {
            kr.store(k);
        }
    };
    fetch(0);
    for (int u = 0; u < count; ++u) {
        __syncthreads();
        put();
        __syncthreads();
        fetch(u + 1);
        const int k0 = (int)list[u] * BA_BLOCK;
        const bool bit = R.mine && ((mask[u] >> R.ql) & 1);
        if constexpr (CAREFUL)
            poison |= bit && (*odd & (R.limit - k0 >= BA_BLOCK ? ~0ull : (1ull << max(0, R.limit - k0)) - 1)) != 0;
        ba_dq_block<T, DP>(a, R, qf, gf, stat, delta, up, k, k0, bit, acc);
    }
}

template <typename T, int DP, bool CAREFUL> __device__ __forceinline__ void ba_dq_tile(const BaArgs &a, int64_t id, char *smem, unsigned long long *odd)
{
    typedef BaLds<T, DP> L;
    typedef typename hd_vec<T>::v8 V8;
    constexpr bool HALF = __is_same(T, _Float16);
    uint64_t *mask = (uint64_t *)(smem + 2 * L::TILE);
    uint32_t *list = (uint32_t *)(mask + a.cap), *words = list + a.cap, *before = words + (a.nb + 31) / 32;

    const BaTile t = ba_tile(a, id);
    const int g = (threadIdx.x & 63) >> 4;
    const BaRow R(a, t);
    V8 qf[DP / 32], gf[DP / 32];
    ba_row_operand<T, DP>(R.at<T>(a.q, t.b), R.mine, a.d, qf);
    ba_row_operand<T, DP>(R.at<T>(a.go, t.b), R.mine, a.d, gf);
    float delta = 0.f, up;
    BaStat stat = {0.f, 0.f};
    {
        // the rounding of o, times a gradient, would move all of a row's ds one way: it goes back in
        V8 of[DP / 32], rf[DP / 32];
        ba_row_operand<T, DP>(R.at<T>(a.o, t.b), R.mine, a.d, of);
        ba_row_operand<T, DP>((const T *)a.rest + R.out(a, t.b), R.mine && a.rest, a.d, rf);
#pragma unroll
        for (int kk = 0; kk < DP / 32; ++kk)
#pragma unroll
            for (int x = 0; x < 8; ++x)
                delta = __builtin_fmaf((float)gf[kk][x], __builtin_fmaf((float)rf[kk][x], 1.f / ba_rest_scale<T>(), (float)of[kk][x]), delta);
        delta = ba_col_sum(delta);
        if (R.mine) {
            const int64_t at = 2 * R.flat(a, t.b);
            stat = {a.lse[at], a.lse[at + 1]};
            if (g == 0)
                a.row[at] = stat.by + (HALF ? BA_P_SHIFT : 0.f), a.row[at + 1] = delta;
        }
    }
    const int count = ba_union(a, t, list, mask, words, before);
    hd_f4 acc[DP / 16];
    bool poison = false;
    ba_dq_pass<T, DP, CAREFUL>(a, t, R, qf, gf, stat, delta, up, smem, mask, list, count, odd, acc, poison);
    auto reached = [&]() __attribute__((always_inline)) {       // this lane's row holds what is not finite
        bool finite = true;
#pragma unroll
        for (int d = 0; d < DP / 16; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                finite &= ba_finite(acc[d][r]);
        return ba_col_max(finite || poison ? 0.f : 1.f) > 0.f;
    };
    if (!CAREFUL && reached())
        atomicOr(a.unclean, 1u);
    if (!R.there)
        return;
    T *O = (T *)a.dq + R.out(a, t.b);
    const float down = poison ? NAN : HALF ? 1.f / up : 1.f;
#pragma unroll
    for (int d = 0; d < DP / 16; ++d)
        if (d * 16 + g * 4 < a.d)
            ba_store4<T>(O + d * 16 + g * 4, acc[d] * down * a.scale);
}

template <typename T, int DP>
__global__ __launch_bounds__(BA_THREADS, (BaBwd<T, DP>::w)) void block_attn_dq_kernel(BaArgs a, int64_t all)
{
    extern __shared__ __attribute__((aligned(16))) char smem[];
    ba_dq_tile<T, DP, false>(a, ba_xcd(blockIdx.x, all), smem, nullptr);
}

// ---- backward: which queries picked a block ------------------------------------------------------------------------------
// bits[(b, h, blk), tile of 64 queries]: a workgroup per (sequence, key head, tile) collects the tile's words in LDS.
constexpr int BP_WORDS = 2048;
__global__ __launch_bounds__(BA_THREADS) void block_pick_bits_kernel(BaArgs a)
{
    __shared__ unsigned long long w[BP_WORDS];
    const int tile = (int)(blockIdx.x % a.mt), bh = (int)(blockIdx.x / a.mt), h = bh % a.hk, b = bh / a.hk;
    const int live = a.n_arr ? min(max(a.n_arr[b], 0), a.n) : a.n, lm = a.m_arr ? min(max(a.m_arr[b], 0), a.m) : a.m;
    const int i0 = tile * 64, entries = min(64, a.m - i0) * a.count;
    if (blockIdx.x == 0 && threadIdx.x == 0)
        *a.unclean = 0;                     // (for the kernels behind this one)
    const int32_t *idx = a.blocks + (((int64_t)b * a.m + i0) * a.hk + h) * a.count;
    for (int b0 = 0; b0 < a.nb; b0 += BP_WORDS) {
        const int words = min(BP_WORDS, a.nb - b0);
        for (int x = threadIdx.x; x < words; x += BA_THREADS)
            w[x] = 0;
        __syncthreads();
        for (int e = threadIdx.x; e < entries; e += BA_THREADS) {
            const int q = e / a.count, blk = idx[(int64_t)q * a.hk * a.count + (e - q * a.count)];
            if (blk >= b0 && blk < b0 + words && blk * BA_BLOCK < ba_limit(a, live, lm, i0 + q))
                atomicOr(w + (blk - b0), 1ull << q);
        }
        __syncthreads();
        for (int x = threadIdx.x; x < words; x += BA_THREADS)
            a.bits[((int64_t)bh * a.nb + b0 + x) * a.mt + tile] = w[x];
        __syncthreads();
    }
}

// Some blocks are picked by many more queries than others (a popular region, the start of a sequence), and where blocks are
// few the chip would wait for the longest.  Their queries are then dealt into parts of `chunk` in order; a part is a
// workgroup's work, and a block of several parts is added up in their order afterwards.
__global__ __launch_bounds__(BA_THREADS) void block_picks_kernel(BaArgs a)
{
    __shared__ int s[4];
    const uint64_t *bits = a.bits + (int64_t)blockIdx.x * a.mt;
    int v = 0;
    for (int w = threadIdx.x; w < a.mt; w += BA_THREADS)
        v += __popcll(bits[w]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        v += __shfl_xor(v, o, 64);
    if ((threadIdx.x & 63) == 0)
        s[threadIdx.x >> 6] = v;
    __syncthreads();
    if (threadIdx.x == 0)
        a.picks[blockIdx.x] = s[0] + s[1] + s[2] + s[3];
}
// first[i] = number of parts of the blocks before i (a block nobody picked is one part: it writes zeros); at most 1024 blocks
__global__ __launch_bounds__(1024) void block_parts_kernel(BaArgs a, int blocks)
{
    __shared__ int s[16];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int mine = t < blocks ? max(1, (a.picks[t] + a.chunk - 1) / a.chunk) : 0;
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(inc, o, 64);
        inc += lane >= o ? v : 0;
    }
    if (lane == 63)
        s[wave] = inc;
    __syncthreads();
    for (int w = 0; w < wave; ++w)
        inc += s[w];
    if (t < blocks)
        a.first[t] = inc - mine;
    if (t == blocks - 1)
        a.first[blocks] = inc;
}

// ---- backward: dk, dv ----------------------------------------------------------------------------------------------------
// A workgroup per block of keys, or per part of the queries that picked it; a wave owns 16 of its keys.  Scores are formed as
// rows x keys here, so that P and dS come out with a key per lane: the B operand of dv^T = do^T P and dk^T = q^T dS.
constexpr int BD_WORDS = 64;                // tiles of queries looked through at a time

// What a workgroup of the dk / dv kernel has: its block, its part of the queries that picked it, in order
struct BaKeys {
    int b, h, live, lm, key;                // key: this lane's
    int skip, take;
    const uint64_t *bits;
};

// CAREFUL: values of q and do that are not finite stay out of the products, and the keys that a row with such a value sees are
// not numbers (poison).
template <typename T, int DP, bool CAREFUL>
__device__ __forceinline__ void ba_dkv_pass(const BaArgs &a, const BaKeys &w, const typename hd_vec<T>::v8 *kf, const typename hd_vec<T>::v8 *vf,
                                            char *smem, int *list_all, unsigned long long *odd,
                                            hd_f4 (&dk)[DP / 16], hd_f4 (&dv)[DP / 16], float &up, bool &poison)
{
    typedef BaLds<T, DP> L;
    typedef typename hd_vec<T>::v8 V8;
    constexpr bool HALF = __is_same(T, _Float16);
    T *Qs = (T *)smem, *Gs = (T *)(smem + L::TILE);
    float *top_s = (float *)(smem + 2 * L::TILE), *by_s = top_s + 64, *delta_s = by_s + 64;
    int *limit_s = (int *)(delta_s + 64), *list = limit_s + 64;              // list: BD_WORDS * 64 queries
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, g = lane >> 4;
    int skip = w.skip, take = w.take;
#pragma unroll
    for (int d = 0; d < DP / 16; ++d)
        dk[d] = dv[d] = hd_f4{0.f, 0.f, 0.f, 0.f};
    up = BA_UP;                             // fp16: this lane's key's ds are taken times this power of two

    typedef BaStage<T, DP> S;
    S qr, gr;
    float row_top = 0.f, row_by = 0.f, row_delta = 0.f;
    int row_limit = 0;
    const T *Q = S::lane((const T *)a.q.data + w.b * a.q.sb + (int64_t)w.h * a.group * a.q.sh, a.d);
    const T *G = S::lane((const T *)a.go.data + w.b * a.go.sb + (int64_t)w.h * a.group * a.go.sh, a.d);
    // rows r0 .. r0 + 63 of the list (query by query, all heads of the group) to registers; rows behind the last are its
    // copies that see nothing
    auto fetch = [&](int r0, int rows) __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < S::PER; ++x) {
            const int r = min(r0 + S::row(x), rows - 1);
            const int q = a.group == 1 ? r : (int)__umulhi((unsigned)r, a.group_inverse), e = r - q * a.group;
            const int64_t i = list[q];
            qr.r[x] = *(const V8 *)(Q + i * a.q.sr + e * a.q.sh);
            gr.r[x] = *(const V8 *)(G + i * a.go.sr + e * a.go.sh);
        }
        row_top = row_by = row_delta = 0.f;
        row_limit = 0;
        if (threadIdx.x < BA_ROWS && r0 + (int)threadIdx.x < rows) {
            const int r = r0 + threadIdx.x, q = r / a.group, head = w.h * a.group + (r - q * a.group), i = list[q];
            const int64_t p = ((int64_t)w.b * a.hq + head) * a.m + i;
            row_top = a.lse[2 * p], row_by = a.row[2 * p], row_delta = a.row[2 * p + 1];
            row_limit = ba_limit(a, w.live, w.lm, i);
        }
    };

    for (int w0 = 0; w0 < a.mt && take > 0; w0 += BD_WORDS) {
        // the queries of the next 64 tiles that picked this block, in order; `skip` of them are other parts', `take` are ours
        if (wave == 0) {
            uint64_t word = w0 + lane < a.mt ? w.bits[w0 + lane] : 0ull;
            int inc = __popcll(word), at = -inc;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int v = __shfl_up(inc, o, 64);
                inc += lane >= o ? v : 0;
            }
            at += inc - skip;
            if (lane == 63)
                *list_all = inc;
            for (; word; word &= word - 1, ++at)
                if (at >= 0 && at < take)
                    list[at] = (w0 + lane) * 64 + __ffsll((unsigned long long)word) - 1;
        }
        __syncthreads();
        const int here = min(take, max(0, *list_all - skip)), rows = here * a.group;
        skip = max(0, skip - *list_all);
        take -= here;
        if (rows > 0)
            fetch(0, rows);
        for (int r0 = 0; r0 < rows; r0 += BA_ROWS) {
            __syncthreads();                // the previous tile has been read
            if constexpr (CAREFUL) {
                if (threadIdx.x == 0)
                    *odd = 0;
                __syncthreads();
                qr.store_finite(Qs, odd);
                gr.store_finite(Gs, odd);
            } else {
                qr.store(Qs);
                gr.store(Gs);
            }
            if (threadIdx.x < BA_ROWS) {
                top_s[threadIdx.x] = row_top, by_s[threadIdx.x] = row_by;
                delta_s[threadIdx.x] = row_delta, limit_s[threadIdx.x] = row_limit;
            }
            __syncthreads();
            if (r0 + BA_ROWS < rows)
                fetch(r0 + BA_ROWS, rows);
            if constexpr (CAREFUL)
                for (unsigned long long left = *odd; left; left &= left - 1)
                    poison |= w.key < limit_s[__ffsll(left) - 1];
#pragma unroll
            for (int j = 0; j < 2; ++j) {   // 32 rows at a time
                hd_f4 p[2], ds[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    V8 qa[DP / 32], ga[DP / 32];
#pragma unroll
                    for (int kk = 0; kk < DP / 32; ++kk) {
                        qa[kk] = L::row8(Qs, j * 32 + x * 16 + l15, kk * 4 + g);
                        ga[kk] = L::row8(Gs, j * 32 + x * 16 + l15, kk * 4 + g);
                    }
                    const int r4 = j * 32 + x * 16 + g * 4;
                    const hd_f4 to = *(const hd_f4 *)(top_s + r4), by = *(const hd_f4 *)(by_s + r4), de = *(const hd_f4 *)(delta_s + r4);
                    const int4 li = *(const int4 *)(limit_s + r4);
                    const int lim[4] = {li.x, li.y, li.z, li.w};
                    ba_issue();
                    hd_f4 s = {0.f, 0.f, 0.f, 0.f}, dp = s;
#pragma unroll
                    for (int kk = 0; kk < DP / 32; ++kk) {
                        s = ba_score_mma<T>(qa[kk], kf[kk], s);
                        dp = ba_score_mma<T>(ga[kk], vf[kk], dp);
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const bool see = w.key < lim[r];
                        const float e = ba_probability<T>(a, s[r], to[r], by[r]);
                        const float f = e * (dp[r] - de[r]);
                        p[x][r] = see ? e : 0.f;
                        ds[x][r] = see ? f : 0.f;
                    }
                }
                if constexpr (HALF) {
                    float big = 0.f;
#pragma unroll
                    for (int x = 0; x < 2; ++x)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            big = fmaxf(big, fabsf(ds[x][r]));
                    ba_lower(ba_col_max(big), up, dk);
                    ds[0] *= up, ds[1] *= up;
                }
                const V8 pf = ba_pack<T>(p[0], p[1]), sf = ba_pack<T>(ds[0], ds[1]);
                // 16-bit types: what their rounding took, as a second term (one term alone: gradients off by 1.4 - 1.6 times
                // what the plain form in 32 bits and its last rounding are off; 72 -> 82 and 365 -> 400 us)
                V8 pr, sr;
                if constexpr (sizeof(T) == 2)
                    pr = ba_rest<T>(p[0], p[1], pf), sr = ba_rest<T>(ds[0], ds[1], sf);
                constexpr int TG = DP / 16 < 4 ? DP / 16 : 4;
#pragma unroll
                for (int d0 = 0; d0 < DP / 16; d0 += TG) {
                    V8 gc[TG], qc[TG];
#pragma unroll
                    for (int d = 0; d < TG; ++d) {
                        gc[d] = L::column(Gs, j * 32, d0 + d);
                        qc[d] = L::column(Qs, j * 32, d0 + d);
                    }
                    ba_issue();
#pragma unroll
                    for (int d = 0; d < TG; ++d) {
                        dv[d0 + d] = ba_mma<T>(gc[d], pf, dv[d0 + d]);
                        dk[d0 + d] = ba_mma<T>(qc[d], sf, dk[d0 + d]);
                    }
                    if constexpr (sizeof(T) == 2) {
#pragma unroll
                        for (int d = 0; d < TG; ++d) {
                            dv[d0 + d] = ba_mma<T>(gc[d], pr, dv[d0 + d]);
                            dk[d0 + d] = ba_mma<T>(qc[d], sr, dk[d0 + d]);
                        }
                    }
                }
            }
        }
        __syncthreads();                    // the list is rebuilt
    }
}

template <typename T, int DP, bool CAREFUL>
__device__ __forceinline__ void ba_dkv_part(const BaArgs &a, int64_t id, char *smem, int *list_all, unsigned long long *odd)
{
    typedef typename hd_vec<T>::v8 V8;
    constexpr bool HALF = __is_same(T, _Float16);
    int64_t part = 0;
    int skip = 0, take = 0x7FFFFFFF, parts = 1;                 // of the queries that picked the block, in order
    if (a.chunk) {
        const int blocks = a.b * a.hk * a.nb;
        part = id;
        if (part >= a.first[blocks])
            return;
        int lo = 0, hi = blocks - 1;        // the last block whose first part is not behind this one
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (a.first[mid] <= part)
                lo = mid;
            else
                hi = mid - 1;
        }
        id = lo;
        parts = a.first[lo + 1] - a.first[lo];
        skip = (int)(part - a.first[lo]) * a.chunk;
        take = a.chunk;
    }
    const int blk = (int)(id % a.nb), bh = (int)(id / a.nb), h = bh % a.hk, b = bh / a.hk;
    const int live = a.n_arr ? min(max(a.n_arr[b], 0), a.n) : a.n, lm = a.m_arr ? min(max(a.m_arr[b], 0), a.m) : a.m;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, g = lane >> 4;
    const int key = blk * BA_BLOCK + wave * 16 + l15;
    V8 kf[DP / 32], vf[DP / 32];
    ba_row_operand<T, DP>((const T *)a.k.data + b * a.k.sb + (int64_t)key * a.k.sr + h * a.k.sh, key < live, a.d, kf);
    ba_row_operand<T, DP>((const T *)a.v.data + b * a.v.sb + (int64_t)key * a.v.sr + h * a.v.sh, key < live, a.d, vf);
    hd_f4 dk[DP / 16], dv[DP / 16];
    const BaKeys w = {b, h, live, lm, key, skip, take, a.bits + ((int64_t)bh * a.nb + blk) * a.mt};
    float up;
    bool poison = false;
    auto reached = [&]() __attribute__((always_inline)) {       // this lane's key holds what is not finite
        bool finite = true;
#pragma unroll
        for (int d = 0; d < DP / 16; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                finite &= ba_finite(dk[d][r]) && ba_finite(dv[d][r]);
        return ba_col_max(finite || poison ? 0.f : 1.f) > 0.f;
    };
    ba_dkv_pass<T, DP, CAREFUL>(a, w, kf, vf, smem, list_all, odd, dk, dv, up, poison);
    if constexpr (CAREFUL) {
        poison = ba_col_max(poison ? 1.f : 0.f) > 0.f;
        if (poison)
#pragma unroll
            for (int d = 0; d < DP / 16; ++d)
                dk[d] = dv[d] = hd_f4{NAN, NAN, NAN, NAN};
    } else if (reached()) {
        atomicOr(a.unclean, 1u);
    }
    // (fp16: probabilities came times 2^BA_P_SHIFT)
    constexpr float P_DOWN = HALF ? 1.f / 32768.f : 1.f;
    const float down = HALF ? P_DOWN / up : 1.f;
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) {
        dk[d] = dk[d] * down * a.scale;
        if (HALF)
            dv[d] *= P_DOWN;
    }
    if (parts > 1) {                        // joined by block_attn_dkv_join_kernel
        float *P = a.part + (part * 2 * BA_BLOCK + wave * 16 + l15) * DP;
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) {
            *(hd_f4 *)(P + d * 16 + g * 4) = dk[d];
            *(hd_f4 *)(P + BA_BLOCK * DP + d * 16 + g * 4) = dv[d];
        }
        return;
    }
    if (key >= a.n)
        return;
    const int64_t at = (((int64_t)b * a.n + key) * a.hk + h) * a.d;
#pragma unroll
    for (int d = 0; d < DP / 16; ++d)
        if (d * 16 + g * 4 < a.d) {
            ba_store4<T>((T *)a.out + at + d * 16 + g * 4, dk[d]);
            ba_store4<T>((T *)a.out2 + at + d * 16 + g * 4, dv[d]);
        }
}

template <typename T, int DP>
__global__ __launch_bounds__(BA_THREADS, (BaBwd<T, DP>::kw)) void block_attn_dkv_kernel(BaArgs a, int64_t all)
{
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ int list_all;
    ba_dkv_part<T, DP, false>(a, ba_xcd(blockIdx.x, all), smem, &list_all, nullptr);
}

// Both once more, carefully, where anything came out that is not finite (a launch that ends at once where nothing did: 4.6 us;
// inside the two kernels above the careful passes cost registers, and with them 388 for 357 us).
template <typename T, int DP> __global__ __launch_bounds__(BA_THREADS) void block_attn_careful_kernel(BaArgs a, int64_t tiles, int64_t parts)
{
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ int list_all;
    __shared__ unsigned long long odd;
    if (!*a.unclean)
        return;
    if (blockIdx.x < tiles)
        ba_dq_tile<T, DP, true>(a, blockIdx.x, smem, &odd);
    else
        ba_dkv_part<T, DP, true>(a, blockIdx.x - tiles, smem, &list_all, &odd);
}

// dk and dv of a block from its parts, in the parts' order
constexpr int BJ_SLICES = 4;                // workgroups a block
template <typename T, int DP> __global__ __launch_bounds__(BA_THREADS) void block_attn_dkv_join_kernel(BaArgs a)
{
    const int id = (int)(blockIdx.x / BJ_SLICES), blk = id % a.nb, bh = id / a.nb, h = bh % a.hk, b = bh / a.hk;
    const int p0 = a.first[id], p1 = a.first[id + 1];
    if (p1 - p0 < 2)
        return;
    constexpr int EACH = 2 * BA_BLOCK * DP / 4 / BJ_SLICES;
    const int e0 = (int)(blockIdx.x % BJ_SLICES) * EACH;
    for (int e = e0 + threadIdx.x; e < e0 + EACH; e += BA_THREADS) {
        const int row = e / (DP / 4), c = (e % (DP / 4)) * 4, key = blk * BA_BLOCK + row % BA_BLOCK;
        if (key >= a.n || c >= a.d)
            continue;
        hd_f4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int p = p0; p < p1; ++p)
            y += *(const hd_f4 *)(a.part + ((int64_t)p * 2 * BA_BLOCK + row) * DP + c);
        T *O = (T *)(row < BA_BLOCK ? a.out : a.out2);
        ba_store4<T>(O + (((int64_t)b * a.n + key) * a.hk + h) * a.d + c, y);
    }
}

// ---- host --------------------------------------------------------------------------------------------------------------
int ba_fill(BaArgs &a, int type, int b, int m, int n, int d, const tpu3_heads *q, const tpu3_heads *k, const tpu3_heads *v,
            const int32_t *blocks, int count, double scale, const int32_t *n_arr, const int32_t *m_arr, int causal)
{
    if (b < 0 || m < 0 || n < 0 || d <= 0 || !hd_type_ok(type) || !q || !k || !v || q->heads <= 0 || k->heads <= 0 ||
        q->heads % k->heads || v->heads != k->heads || count <= 0 || !(scale >= 1e-30) || scale > 1e30)
        return TPU3_EINVAL;
    if (d % 8 || d > 128 || count > TPU3_BLOCK_COUNT_MAX || q->heads / k->heads > BA_ROWS ||
        (n > 0 && (n - 1) / BA_BLOCK + 1 > TPU3_ATTN_BLOCKS_MAX))
        return TPU3_ELIMIT;
    a.q = *q, a.k = *k, a.v = *v, a.blocks = blocks, a.n_arr = n_arr, a.m_arr = m_arr;
    a.b = b, a.m = m, a.n = n, a.nb = n > 0 ? (n - 1) / BA_BLOCK + 1 : 0, a.mt = m > 0 ? (m - 1) / 64 + 1 : 0;
    a.hq = q->heads, a.hk = k->heads, a.group = a.hq / a.hk, a.d = d, a.count = count, a.causal = causal != 0;
    a.scale = (float)scale, a.scale2 = (float)(scale * 1.44269504088896340736);
    if (type == TPU3_TYPE_F32 && (double)a.scale2 >= scale * 1.44269504088896340736)
        a.scale2 = nextafterf(a.scale2, 0.f);                   // (the rest above 0: a masked score times it stays -infinity)
    a.scale2_rest = (float)(scale * 1.44269504088896340736 - (double)a.scale2);
    a.group_inverse = a.group > 1 ? (unsigned)(((1ull << 32) + a.group - 1) / a.group) : 0u;
    a.qt = BA_ROWS / a.group;
    a.tiles = m > 0 ? (m - 1) / a.qt + 1 : 0;
    a.cap = a.qt * count < a.nb ? a.qt * count : a.nb;
    a.splits = 1;
    if (b == 0 || m == 0)
        return TPU3_OK;
    if (!hd_rows_ok(q, type) || !blocks || (n > 0 && (!hd_rows_ok(k, type) || !hd_rows_ok(v, type))))
        return TPU3_EINVAL;
    const int64_t most = (1 << 23) - 1;     // workgroups of 256 threads: 2^32 threads a launch, two kinds of them in one
    if ((int64_t)b * a.hk * a.tiles > most || (int64_t)b * a.hk * a.nb > most || (int64_t)b * a.hk * a.mt > most)
        return TPU3_ELIMIT;
    return 1;
}

// Splits of a tile's blocks where the tiles alone do not fill the chip: up to four workgroups a compute unit, two for single
// tokens (their blocks are few, and the join reads every split), and about one block a split.  Measured, us with / without:
// 8 sequences, one token of 32 over 8 heads of 128 channels, 16 blocks: 15 / 25; the same for 8 tokens: 18 / 26; 312 tiles
// of 32 queries whose picks differ (24 channels, 5 blocks each): 55 / 87.  From 512 tiles on it does not pay: 42 / 27.
int ba_splits(int b, int m, int n, int hq, int hk, int count)
{
    if (b <= 0 || m <= 0 || n <= 0 || hk <= 0 || hq < hk || count <= 0)
        return 1;
    const int qt = BA_ROWS / (hq / hk);
    if (qt < 1)
        return 1;
    const int64_t tiles = (int64_t)b * hk * ((m - 1) / qt + 1), used = (int64_t)(m < qt ? m : qt) * count, nb = (n - 1) / BA_BLOCK + 1;
    if (tiles >= 512)
        return 1;
    int64_t s = (m <= 16 ? 512 : 1024) / tiles;
    s = s < used ? s : used;
    s = s < nb ? s : nb;
    s = s < 2 * count ? s : 2 * count;
    return s < 1 ? 1 : s > 64 ? 64 : (int)s;
}

// Queries of a part of the dk / dv pass where blocks are few (0: a workgroup per block), and the most parts there can be.
// Measured, us for forward and backward with parts / a workgroup per block: 128 blocks (2048 queries, 8 heads over 2, 64
// channels, 8 blocks each): 82 / 116, and 82 / 215 where all pick the first; 1024 blocks (8192 queries, 8 heads): 182 / 147,
// and 186 / 256 where all pick the first, which is what the parts are for.  Where no block can have more than four parts, and
// there are enough blocks for the chip, they only cost: 960 blocks (48 sequences of 312, 4 heads): 99 / 73.
int ba_dkv_chunk(int b, int m, int hk, int nb, int count)
{
    const int64_t blocks = (int64_t)b * hk * nb;
    if (blocks <= 0 || blocks > 1024)
        return 0;
    const int64_t picks = (int64_t)b * hk * m * (count < nb ? count : nb);
    int64_t c = (picks / 1024 + 63) / 64 * 64;
    c = c < 128 ? 128 : c;
    return blocks > 256 && m <= 4 * c ? 0 : (int)c;
}
int64_t ba_dkv_parts(int b, int m, int hk, int nb, int count)
{
    const int64_t picks = (int64_t)b * hk * m * (count < nb ? count : nb);
    return (int64_t)b * hk * nb + picks / ba_dkv_chunk(b, m, hk, nb, count);
}

int ba_dp(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }

size_t ba_lds(const BaArgs &a, size_t tiles) { return tiles + (size_t)a.cap * 12 + (size_t)((a.nb + 31) / 32) * 8; }

// The most that a launch of any size needs, the same in every call: calls from several threads do not change each other's limit
// between setting it and launching.
template <typename T, int DP> constexpr size_t ba_lds_most()
{
    return 2 * BaLds<T, DP>::TILE + (size_t)BA_ROWS * TPU3_BLOCK_COUNT_MAX * 12 + TPU3_ATTN_BLOCKS_MAX / 32 * 8;
}
template <typename T, int DP, typename K> int ba_allow(K kernel)
{
    return (int)hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)ba_lds_most<T, DP>());
}

template <typename T, int DP> int ba_forward(const BaArgs &a, hipStream_t s)
{
    const int64_t all = (int64_t)a.b * a.hk * a.tiles * a.splits;
    const size_t lds = ba_lds(a, 2 * BaLds<T, DP>::TILE);
    int rc = ba_allow<T, DP>(block_attn_fwd_kernel<T, DP>);
    if (rc)
        return rc;
    hipLaunchKernelGGL((block_attn_fwd_kernel<T, DP>), dim3((unsigned)all), dim3(BA_THREADS), lds, s, a, all);
    if (a.splits > 1) {
        const int64_t rows = (int64_t)a.b * a.hq * a.m, per = BA_THREADS / (a.splits <= 16 ? 16 : 64);
        const dim3 grid((unsigned)((rows + per - 1) / per));
        if (a.splits <= 16)
            hipLaunchKernelGGL((block_attn_join_kernel<T, DP, 16>), grid, dim3(BA_THREADS), 0, s, a, rows);
        else
            hipLaunchKernelGGL((block_attn_join_kernel<T, DP, 64>), grid, dim3(BA_THREADS), 0, s, a, rows);
    }
    return tpu3_launch_status();
}

template <typename T, int DP> int ba_backward(BaArgs a, void *dq, void *dk, void *dv, hipStream_t s)
{
    const int64_t tiles = (int64_t)a.b * a.hk * a.tiles, blocks = (int64_t)a.b * a.hk * a.nb;
    const int64_t parts = a.chunk ? ba_dkv_parts(a.b, a.m, a.hk, a.nb, a.count) : blocks;
    const size_t lds = ba_lds(a, 2 * BaLds<T, DP>::TILE), lds2 = 2 * BaLds<T, DP>::TILE + 4 * 64 * 4 + (size_t)BD_WORDS * 64 * 4;
    const size_t most = lds > lds2 ? lds : lds2;
    static_assert(2 * BaLds<T, DP>::TILE + 4 * 64 * 4 + (size_t)BD_WORDS * 64 * 4 <= ba_lds_most<T, DP>(), "");
    int rc = ba_allow<T, DP>(block_attn_dq_kernel<T, DP>);
    if (!rc)
        rc = ba_allow<T, DP>(block_attn_dkv_kernel<T, DP>);
    if (!rc)
        rc = ba_allow<T, DP>(block_attn_careful_kernel<T, DP>);
    if (rc)
        return rc;
    a.dq = dq, a.out = dk, a.out2 = dv;
    hipLaunchKernelGGL(block_pick_bits_kernel, dim3((unsigned)(a.b * a.hk * a.mt)), dim3(BA_THREADS), 0, s, a);
    // dq also leaves the rows' do . o for the pass over the keys
    hipLaunchKernelGGL((block_attn_dq_kernel<T, DP>), dim3((unsigned)tiles), dim3(BA_THREADS), lds, s, a, tiles);
    if (a.nb == 0)
        return tpu3_launch_status();
    if (a.chunk) {
        hipLaunchKernelGGL(block_picks_kernel, dim3((unsigned)blocks), dim3(BA_THREADS), 0, s, a);
        hipLaunchKernelGGL(block_parts_kernel, dim3(1), dim3(1024), 0, s, a, (int)blocks);
    }
    hipLaunchKernelGGL((block_attn_dkv_kernel<T, DP>), dim3((unsigned)parts), dim3(BA_THREADS), lds2, s, a, parts);
    hipLaunchKernelGGL((block_attn_careful_kernel<T, DP>), dim3((unsigned)(tiles + parts)), dim3(BA_THREADS), most, s, a, tiles, parts);
    if (a.chunk)
        hipLaunchKernelGGL((block_attn_dkv_join_kernel<T, DP>), dim3((unsigned)(blocks * BJ_SLICES)), dim3(BA_THREADS), 0, s, a);
    return tpu3_launch_status();
}

template <typename T> int ba_forward_d(const BaArgs &a, hipStream_t s)
{
    const int dp = ba_dp(a.d);
    return dp == 32 ? ba_forward<T, 32>(a, s) : dp == 64 ? ba_forward<T, 64>(a, s) : ba_forward<T, 128>(a, s);
}
template <typename T> int ba_backward_d(const BaArgs &a, void *dq, void *dk, void *dv, hipStream_t s)
{
    const int dp = ba_dp(a.d);
    return dp == 32 ? ba_backward<T, 32>(a, dq, dk, dv, s) : dp == 64 ? ba_backward<T, 64>(a, dq, dk, dv, s) : ba_backward<T, 128>(a, dq, dk, dv, s);
}

}  // namespace

extern "C" size_t tpu3_block_attn_fwd_workspace_bytes(int b, int m, int n, int hq, int hk, int d, int count)
{
    const int s = ba_splits(b, m, n, hq, hk, count);
    return s == 1 ? 0 : (size_t)b * m * hq * s * (ba_dp(d) + 4) * 4;
}

extern "C" int tpu3_block_attn_fwd(tpu3_stream_t stream, int type, int b, int m, int n, int d, const tpu3_heads *q,
                                   const tpu3_heads *k, const tpu3_heads *v, const int32_t *blocks, int count, double scale,
                                   const int32_t *n_arr, const int32_t *m_arr, int causal, void *out, float *lse,
                                   void *rest, void *workspace, size_t workspace_bytes)
{
    BaArgs a = {};
    const int rc = ba_fill(a, type, b, m, n, d, q, k, v, blocks, count, scale, n_arr, m_arr, causal);
    if (rc <= 0)
        return rc;
    if (!out || ((uintptr_t)out & 15) || ((uintptr_t)rest & 15) || ((uintptr_t)lse & 7))
        return TPU3_EINVAL;
    a.out = out, a.lse = lse, a.rest = type == TPU3_TYPE_F32 ? nullptr : rest;
    a.splits = ba_splits(b, m, n, a.hq, a.hk, count);
    if (a.splits > 1) {
        if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < (size_t)b * m * a.hq * a.splits * (ba_dp(d) + 4) * 4)
            return TPU3_EINVAL;
        a.part = (float *)workspace;
    }
    const hipStream_t s = (hipStream_t)stream;
    return type == TPU3_TYPE_F32 ? ba_forward_d<float>(a, s) : type == TPU3_TYPE_F16 ? ba_forward_d<_Float16>(a, s) : ba_forward_d<__bf16>(a, s);
}

namespace {
// the pieces of the backward workspace: bits, row, unclean, picks, first, part
struct BaBwdLayout {
    size_t row, unclean, picks, first, part, bytes;
};
BaBwdLayout ba_bwd_layout(int b, int m, int n, int hq, int hk, int d, int count)
{
    const size_t nb = n > 0 ? (size_t)(n - 1) / BA_BLOCK + 1 : 0, mt = ((size_t)m + 63) / 64, blocks = (size_t)b * hk * nb;
    const bool parts = ba_dkv_chunk(b, m, hk, (int)nb, count) > 0;
    auto up = [](size_t x) { return (x + 15) / 16 * 16; };
    BaBwdLayout l;
    l.row = up(blocks * mt * 8);
    l.unclean = l.row + up((size_t)b * hq * m * 8);
    l.picks = l.unclean + 16;
    l.first = l.picks + (parts ? up(blocks * 4) : 0);
    l.part = l.first + (parts ? up((blocks + 1) * 4) : 0);
    l.bytes = l.part + (parts ? (size_t)ba_dkv_parts(b, m, hk, (int)nb, count) * 2 * BA_BLOCK * ba_dp(d) * 4 : 0);
    return l;
}
}  // namespace

extern "C" size_t tpu3_block_attn_bwd_workspace_bytes(int b, int m, int n, int hq, int hk, int d, int count)
{
    if (b <= 0 || m <= 0 || hq <= 0 || hk <= 0 || d <= 0 || count <= 0)
        return 0;
    return ba_bwd_layout(b, m, n, hq, hk, d, count).bytes;
}

extern "C" int tpu3_block_attn_bwd(tpu3_stream_t stream, int type, int b, int m, int n, int d, const tpu3_heads *q,
                                   const tpu3_heads *k, const tpu3_heads *v, const tpu3_heads *o, const tpu3_heads *go,
                                   const int32_t *blocks, int count, double scale, const int32_t *n_arr, const int32_t *m_arr,
                                   int causal, const float *lse, const void *rest, void *dq, void *dk, void *dv,
                                   void *workspace, size_t workspace_bytes)
{
    BaArgs a = {};
    const int rc = ba_fill(a, type, b, m, n, d, q, k, v, blocks, count, scale, n_arr, m_arr, causal);
    if (rc <= 0)
        return rc;
    if (!hd_rows_ok(o, type) || !hd_rows_ok(go, type) || o->heads != a.hq || go->heads != a.hq || !lse || ((uintptr_t)lse & 7) || !dq || ((uintptr_t)rest & 15) ||
        ((uintptr_t)dq & 15) || (n > 0 && (!dk || !dv || ((uintptr_t)dk & 15) || ((uintptr_t)dv & 15))) || !workspace ||
        ((uintptr_t)workspace & 15) || workspace_bytes < tpu3_block_attn_bwd_workspace_bytes(b, m, n, a.hq, a.hk, d, count))
        return TPU3_EINVAL;
    a.o = *o, a.go = *go, a.lse = (float *)lse, a.rest = type == TPU3_TYPE_F32 ? nullptr : (void *)rest;
    const BaBwdLayout l = ba_bwd_layout(b, m, n, a.hq, a.hk, d, count);
    a.chunk = ba_dkv_chunk(b, m, a.hk, a.nb, count);
    a.bits = (uint64_t *)workspace;
    a.row = (float *)((char *)workspace + l.row);
    a.unclean = (uint32_t *)((char *)workspace + l.unclean);
    a.picks = (int32_t *)((char *)workspace + l.picks);
    a.first = (int32_t *)((char *)workspace + l.first);
    a.part = (float *)((char *)workspace + l.part);
    const hipStream_t s = (hipStream_t)stream;
    return type == TPU3_TYPE_F32 ? ba_backward_d<float>(a, dq, dk, dv, s) : type == TPU3_TYPE_F16 ? ba_backward_d<_Float16>(a, dq, dk, dv, s) : ba_backward_d<__bf16>(a, dq, dk, dv, s);
}
