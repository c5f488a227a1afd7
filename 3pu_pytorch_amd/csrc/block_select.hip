// block_select.hip -- the cheap score that picks, for every query, which blocks of 64 consecutive keys it attends to.
//
//   mean[b]     = mean of the block's live key rows, per key head                      (tpu3_block_means)
//   score[i, b] = (sum over the heads of the group of q_i) . mean[b]                   (tpu3_block_select)
//   picked      = the `count` best scores, equal ones to the lowest block, listed in ascending order, -1 behind them
//   causal      : position p = n - m + i; the block that holds p always, the rest among the blocks before it (complete
//                 ones: a mean over rows that the query must not see would leak)
//
// The scores are formed in 64 bits: their ORDER decides which keys are read, so two blocks whose scores differ by less
// than an fp32 rounding must not change places with the order of a sum.  A product of two fp32 numbers is exact in 64
// bits, and the sums round 2^29 times finer than fp32's.
#include "heads.h"

namespace {

constexpr int BS_BLOCK = TPU3_ATTN_BLOCK;
constexpr int BS_THREADS = 256;

// ---- means -------------------------------------------------------------------------------------------------------------
// A workgroup per (sequence, block): a thread adds up eight channels over a part of the block's 64 rows, the parts meet in
// LDS in a fixed order.  Bound by reading the keys once.
template <typename T>
__global__ __launch_bounds__(BS_THREADS) void block_means_kernel(int n, int d, int nb, int blocks, int last, tpu3_heads k,
                                                                const int32_t *__restrict__ n_arr, float *__restrict__ means)
{
    __shared__ double red[BS_THREADS * 8];
    const int b = blockIdx.x / blocks, j = blockIdx.x - b * blocks;
    const int live = n_arr ? min(max(n_arr[b], 0), n) : n;
    // all blocks, or those that hold one of the `last` newest rows
    const int blk = j + (last >= 0 ? max(0, live - last) / BS_BLOCK : 0);
    if (blk >= nb || (last >= 0 && blk * BS_BLOCK >= live))
        return;
    const int rows = min(BS_BLOCK, live - blk * BS_BLOCK);
    const int chunks = k.heads * (d / 8);
    float *M = means + ((int64_t)b * nb + blk) * k.heads * d;
    const T *K = (const T *)k.data + b * k.sb + (int64_t)blk * BS_BLOCK * k.sr;
    for (int c0 = 0; c0 < chunks; c0 += BS_THREADS) {
        const int here = min(chunks - c0, BS_THREADS);
        const int parts = here > 128 ? 1 : here > 64 ? 2 : here > 32 ? 4 : 8, per = BS_BLOCK / parts;
        const int part = threadIdx.x / here, c = threadIdx.x - part * here;
        double s[8] = {};
        if (part < parts) {
            const int h = (c0 + c) / (d / 8), ch = ((c0 + c) - h * (d / 8)) * 8;
            const T *src = K + h * k.sh + ch;
            const int r1 = min(rows, (part + 1) * per);
#pragma unroll 4
            for (int r = part * per; r < r1; ++r) {
                float x[8];
                hd_load8(src + r * k.sr, x);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    s[i] += (double)x[i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                red[(part * here + c) * 8 + i] = s[i];
        }
        __syncthreads();
        if (part == 0) {
            for (int p = 1; p < parts; ++p)
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    s[i] += red[(p * here + c) * 8 + i];
            const double inv = rows > 0 ? (double)rows : 1.0;
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                y[i] = (float)(s[i] / inv);
            hd_store8(M + (c0 + c) * 8, y);
        }
        __syncthreads();
    }
}

// ---- selection ---------------------------------------------------------------------------------------------------------
struct BsArgs {
    tpu3_heads q;
    const float *means;
    const int32_t *n_arr, *m_arr;
    int32_t *out;                           // (b, m, hk, count)
    uint64_t *ws_key;                       // (b, hk, m, splits, count)
    int32_t *ws_id;
    uint64_t *open;                         // block_select_many_kernel: queries left open, a word of 64 a wave
    int b, m, n, nb, hk, group, d, count, causal, splits;
};

constexpr int BS_KEEP = 1024;               // candidates in LDS at a time
constexpr int BS_MAX = TPU3_BLOCK_COUNT_MAX;

// Scores as unsigned numbers of the same order (0 is below every score: no candidate).
__device__ __forceinline__ uint64_t bs_key(double v)
{
    if (!(v == v))
        v = -INFINITY;                      // not a number: behind every number
    v += 0.0;                               // -0 is 0
    const uint64_t u = (uint64_t)__double_as_longlong(v);
    return u ^ ((u >> 63) ? ~0ull : 0x8000000000000000ull);
}
constexpr uint64_t BS_OWN = ~0ull;          // above every score: the block that a causal query always gets

struct BsShared {
    double q[128];
    uint64_t key[BS_KEEP];
    int id[BS_KEEP];
    uint64_t wave_key[4 * BS_MAX];
    int wave_id[4 * BS_MAX];
};

__device__ __forceinline__ bool bs_better(uint64_t a, int ia, uint64_t b, int ib) { return a > b || (a == b && ia < ib); }

// The `count` best of the n candidates in s.key / s.id, best first, into their first places; the rest of these places is
// filled with (0, INT_MAX).  A lane sorts its four candidates once; its wave then takes the best head `count` times, by the
// keys' upper halves and, only where these are equal, by the lower halves and the ids.  The waves' lists meet by rank.
__device__ void bs_best(BsShared &s, int n, int count)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool one = n <= 256;              // one wave holds them all
    uint64_t v[4];
    int id[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int e = one ? (wave ? n : j * 64 + lane) : j * BS_THREADS + threadIdx.x;
        v[j] = e < n ? s.key[e] : 0ull;
        id[j] = e < n ? s.id[e] : 0x7FFFFFFF;
    }
    auto order = [&](int x, int y) __attribute__((always_inline)) {
        if (bs_better(v[y], id[y], v[x], id[x])) {
            const uint64_t t = v[x];
            const int u = id[x];
            v[x] = v[y], id[x] = id[y];
            v[y] = t, id[y] = u;
        }
    };
    order(0, 1), order(2, 3), order(0, 2), order(1, 3), order(1, 2);
    for (int r = 0; r < (one && wave ? 0 : count); ++r) {
        const uint32_t hi = (uint32_t)(v[0] >> 32), lo = (uint32_t)v[0];
        const uint32_t mh = tpu3_wave_max_u32(hi);
        unsigned long long who = __ballot(hi == mh);
        if (__popcll(who) > 1) {
            const uint32_t ml = tpu3_wave_max_u32(hi == mh ? lo : 0u);
            who = __ballot(hi == mh && lo == ml);
            if (__popcll(who) > 1) {
                const uint32_t mi = tpu3_wave_min_u32(hi == mh && lo == ml ? (uint32_t)id[0] : 0xFFFFFFFFu);
                who = __ballot(hi == mh && lo == ml && (uint32_t)id[0] == mi);
            }
        }
        if (lane == __ffsll(who) - 1) {
            if (one)
                s.key[r] = v[0], s.id[r] = id[0];               // (all of them are in registers)
            else
                s.wave_key[wave * count + r] = v[0], s.wave_id[wave * count + r] = id[0];
#pragma unroll
            for (int j = 0; j < 3; ++j)
                v[j] = v[j + 1], id[j] = id[j + 1];
            v[3] = 0ull, id[3] = 0x7FFFFFFF;
        }
    }
    __syncthreads();
    if (one)
        return;
    const int c = threadIdx.x;              // 4 * count <= 256 candidates, one a thread
    if (c < 4 * count) {
        const uint64_t cv = s.wave_key[c];
        const int ci = s.wave_id[c];
        int rank = 0;
#pragma unroll 8
        for (int o = 0; o < 4 * count; ++o) {
            const uint64_t ov = s.wave_key[o];
            const int oi = s.wave_id[o];
            rank += bs_better(ov, oi, cv, ci) || (ov == cv && oi == ci && o < c) ? 1 : 0;
        }
        if (rank < count)
            s.key[rank] = cv, s.id[rank] = ci;
    }
    __syncthreads();
}

// ascending ids of the first `count` places (INT_MAX: none) to out, -1 behind them
__device__ void bs_emit(const BsShared &s, int count, int32_t *out)
{
    const int t = threadIdx.x;
    if (t < count) {
        const int me = s.id[t];
        int rank = 0;
        for (int o = 0; o < count; ++o)
            rank += s.id[o] < me || (s.id[o] == me && o < t) ? 1 : 0;
        out[rank] = me == 0x7FFFFFFF ? -1 : me;
    }
}

// A workgroup per (query, key head, part of the blocks).  Eight lanes form a score: each adds up every eighth group of four
// channels, three exchanges join them.
template <typename T, int DP> __device__ void block_select_row(const BsArgs &a, BsShared &s, int64_t row, int z)
{
    const int i = (int)(row % a.m);
    const int bh = (int)(row / a.m), h = bh % a.hk, b = bh / a.hk;
    const int live = a.n_arr ? min(max(a.n_arr[b], 0), a.n) : a.n, lm = a.m_arr ? min(max(a.m_arr[b], 0), a.m) : a.m;
    int end = (live + BS_BLOCK - 1) / BS_BLOCK, own = -1;       // blocks [0, end) are candidates
    if (a.causal) {
        const int p = live - lm + i;
        own = p >= 0 ? p / BS_BLOCK : -1;
        end = own + 1;
    }
    if (i >= lm)
        end = 0;
    const int per = (a.nb + a.splits - 1) / a.splits, z0 = min(end, z * per), z1 = min(end, z0 + per);
    int32_t *out = a.out + (((int64_t)b * a.m + i) * a.hk + h) * a.count;
    const T *Q = (const T *)a.q.data + b * a.q.sb + i * a.q.sr + (int64_t)h * a.group * a.q.sh;
    for (int c = threadIdx.x; c < 128; c += BS_THREADS) {
        double v = 0.0;
        if (c < a.d && z1 > z0)
            for (int g = 0; g < a.group; g += 4) {              // (loads of four heads in flight)
                float x[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    x[e] = g + e < a.group ? (float)Q[(g + e) * a.q.sh + c] : 0.f;
                v += ((double)x[0] + (double)x[1]) + ((double)x[2] + (double)x[3]);
            }
        s.q[c] = v;
    }
    __syncthreads();
    const int slot = threadIdx.x >> 3, part = threadIdx.x & 7;
    constexpr int STEP = BS_THREADS / 8, VECS = DP / 32;
    double q[VECS][4];
#pragma unroll
    for (int x = 0; x < VECS; ++x)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            q[x][j] = s.q[x * 32 + part * 4 + j];
    const float *M = a.means + ((int64_t)b * a.nb * a.hk + h) * a.d + part * 4;
    const int64_t stride = (int64_t)a.hk * a.d;
    int kept = 0;                                               // candidates in LDS
    for (int c0 = z0; c0 < z1 || c0 == z0;) {
        const int take = min(z1 - c0, BS_KEEP - kept);
        constexpr int AHEAD = 16 / VECS > 4 ? 4 : 16 / VECS;     // blocks of a lane in flight
        for (int t0 = 0; t0 < take; t0 += AHEAD * STEP) {
            hd_f4 m[AHEAD][VECS];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
#pragma unroll
                for (int x = 0; x < VECS; ++x)
                    m[u][x] = t0 + u * STEP + slot < take && x * 32 + part * 4 < a.d
                                  ? *(const hd_f4 *)(M + (c0 + t0 + u * STEP + slot) * stride + x * 32)
                                  : hd_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int t = t0 + u * STEP + slot, blk = c0 + t;
                double v = 0.0;
#pragma unroll
                for (int x = 0; x < VECS; ++x)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        v = __builtin_fma((double)m[u][x][j], q[x][j], v);
#pragma unroll
                for (int o = 4; o > 0; o >>= 1)
                    v += __shfl_xor(v, o, 64);
                if (t < take && part == 0) {
                    s.key[kept + t] = blk == own ? BS_OWN : bs_key(v);
                    s.id[kept + t] = blk;
                }
            }
        }
        __syncthreads();
        bs_best(s, kept + max(take, 0), a.count);
        kept = a.count;
        c0 += max(take, 1);
    }
    if (a.splits == 1) {
        bs_emit(s, a.count, out);
        return;
    }
    if ((int)threadIdx.x < a.count) {
        const int64_t at = (row * a.splits + z) * a.count + threadIdx.x;
        a.ws_key[at] = s.key[threadIdx.x];
        a.ws_id[at] = s.id[threadIdx.x];
    }
}

template <typename T, int DP> __global__ __launch_bounds__(BS_THREADS) void block_select_kernel(BsArgs a)
{
    __shared__ BsShared s;
    block_select_row<T, DP>(a, s, blockIdx.x / a.splits, (int)(blockIdx.x % a.splits));
}

// The queries that block_select_many_kernel left open: one word of 64 queries a wave of it.  A workgroup looks at quarters of
// words, 16 queries each, every gridDim.x-th: where all are open (equal means throughout) they still spread over the chip.
constexpr int BO_PARTS = 4, BO_QUERIES = 64 / BO_PARTS;
template <typename T, int DP> __global__ __launch_bounds__(BS_THREADS) void block_select_open_kernel(BsArgs a, int qtiles, int64_t waves)
{
    __shared__ BsShared s;
    __shared__ uint32_t open[BS_THREADS];
    const int64_t units = waves * BO_PARTS, step = gridDim.x;
    for (int64_t u0 = blockIdx.x; u0 < units; u0 += step * BS_THREADS) {
        const int64_t u = u0 + threadIdx.x * step;
        const uint32_t mine = u < units ? (uint32_t)(a.open[u / BO_PARTS] >> (u % BO_PARTS * BO_QUERIES)) & ((1u << BO_QUERIES) - 1) : 0u;
        if (!__syncthreads_or(mine != 0))
            continue;
        open[threadIdx.x] = mine;
        __syncthreads();
        for (int t = 0; t < BS_THREADS; ++t)
            for (uint32_t left = open[t]; left; left &= left - 1) {
                const int64_t at = u0 + t * step, w = at / BO_PARTS;
                block_select_row<T, DP>(a, s, w / qtiles * a.m + w % qtiles * 64 + at % BO_PARTS * BO_QUERIES + __ffs(left) - 1, 0);
                __syncthreads();
            }
        __syncthreads();
    }
}

__global__ __launch_bounds__(BS_THREADS) void block_select_join_kernel(BsArgs a)
{
    __shared__ BsShared s;
    const int64_t row = blockIdx.x;
    const int i = (int)(row % a.m);
    const int bh = (int)(row / a.m), h = bh % a.hk, b = bh / a.hk;
    const int all = a.splits * a.count;                         // <= BS_KEEP by the host's choice of splits
    for (int t = threadIdx.x; t < all; t += BS_THREADS) {
        s.key[t] = a.ws_key[row * all + t];
        s.id[t] = a.ws_id[row * all + t];
    }
    __syncthreads();
    bs_best(s, all, a.count);
    bs_emit(s, a.count, a.out + (((int64_t)b * a.m + i) * a.hk + h) * a.count);
}

// ---- selection for many queries ------------------------------------------------------------------------------------------
// A lane per query, 64 queries of one key head a wave.  The scores come from the matrix cores, approximately, with a bound:
// queries and means as two bf16 terms each (hi + lo, |x - hi - lo| <= 2^-18 |x|), three of the four partial products, fp32
// sums: off by at most  eps = (3 * 2^-18 + 3 d 2^-23) |q| max_b |mean_b|  (the terms left out; every addition cut off at
// 2^-23 of what it adds up).  bf16 queries of one head are their own first term: (2^-18 + 2 d 2^-23).  The kernel keeps the
// k + 1 largest scores of every query, a chain of v_med3 (one instruction an entry).  Where the k-th is more than 2 eps above
// the next, the order of the exact scores around that place is known.  For the other queries (a few in a hundred) the wave
// forms the scores of the blocks within 2 eps of the place in 64 bits, one block at a time, to choose among them.  Only where
// these are too many for the list (rows of equal means) or a value is not finite is the query left open to
// block_select_open_kernel.
// IDS, for up to 16 places among up to 1024 blocks: the block's number stands in the score's lowest bits, and the list holds
// four places more, for near ones.  Otherwise a second pass forms the same scores again and lists what is above the place or
// near it (8 clouds of 5000 points, 8 heads of 64 channels, 8 of 79 blocks: 60 us in two passes, 52 in one; 46 since the
// bound counts the channels instead of standing at 2^-13).
constexpr int BT_MORE = 16;                 // places behind `count` for blocks near the edge
constexpr int BT_NEAR = 1 << 30;            // marks them
constexpr int BT_EXTRA = 4;                 // with numbers: places behind the k + 1st
constexpr int BT_STRIDE = 20;               // floats between two queries' 16 scores in LDS

// LDS accesses above and below stay there: between the lanes of one wave nothing more is needed (they complete in order)
__device__ __forceinline__ void bt_exchange()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

struct BtSplit {
    hd_bf8 hi, lo;
};
__device__ __forceinline__ BtSplit bt_split(const float *x)
{
    BtSplit r;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const __bf16 h = (__bf16)x[i];
        r.hi[i] = h;
        r.lo[i] = (__bf16)(x[i] - (float)h);
    }
    return r;
}

template <typename T, int DP, int NL, bool LOQ, bool IDS>
__global__ __launch_bounds__(BS_THREADS) void block_select_many_kernel(BsArgs a, int qtiles, int64_t waves)
{
    constexpr int EXTRA = IDS ? BT_EXTRA : 0;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, g = lane >> 4;
    float *sc = (float *)smem + wave * (64 * BT_STRIDE);
    const int places = IDS ? max(NL, a.count) : max(a.count, min(a.count + BT_MORE, 64));
    int *found = (int *)((float *)smem + 4 * 64 * BT_STRIDE) + wave * 64 * places;          // (places, 64)
    const int64_t w = (int64_t)blockIdx.x * 4 + wave;
    if (w >= waves)
        return;                             // (no barriers below: a wave works by itself)
    const int qt = (int)(w % qtiles), bh = (int)(w / qtiles), h = bh % a.hk, b = bh / a.hk, i0 = qt * 64;
    const int live = a.n_arr ? min(max(a.n_arr[b], 0), a.n) : a.n, lm = a.m_arr ? min(max(a.m_arr[b], 0), a.m) : a.m;
    const int i = i0 + lane;
    int end = (live + BS_BLOCK - 1) / BS_BLOCK, own = -1;       // this lane's query scores the blocks [0, end)
    if (a.causal) {
        const int p = live - lm + i;
        own = i < lm && p >= 0 ? p / BS_BLOCK : -1;
        end = max(own, 0);
    }
    if (i >= lm)
        end = 0;
    const int k = a.count - a.causal;       // wanted among them
    int most = end;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        most = max(most, __shfl_xor(most, o, 64));

    // B operands: rows i0 + sub*16 + l15, channels kk*32 + g*8 .. +8, summed over the group's heads
    BtSplit q[4][DP / 32];
    float qn = 0.f, qp = 0.f;               // |q|^2 of query `lane`; the same of its heads before they are added up, together
    const T *Q = (const T *)a.q.data + b * a.q.sb + (int64_t)h * a.group * a.q.sh;
#pragma unroll
    for (int sub = 0; sub < 4; ++sub) {
        const int r = i0 + sub * 16 + l15;
        float n2 = 0.f, parts = 0.f;
#pragma unroll
        for (int kk = 0; kk < DP / 32; ++kk) {
            const int c = kk * 32 + g * 8;
            float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (r < lm && c < a.d)
                for (int e = 0; e < a.group; ++e) {
                    float y[8];
                    hd_load8(Q + r * a.q.sr + e * a.q.sh + c, y);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        x[j] += y[j];
                        parts = __builtin_fmaf(y[j], y[j], parts);
                    }
                }
#pragma unroll
            for (int j = 0; j < 8; ++j)
                n2 = __builtin_fmaf(x[j], x[j], n2);
            q[sub][kk] = bt_split(x);
        }
        n2 += __shfl_xor(n2, 16, 64);
        n2 += __shfl_xor(n2, 32, 64);
        qn = g == sub ? n2 : qn;            // lane sub*16 + l15
        if (a.group > 1) {
            parts += __shfl_xor(parts, 16, 64);
            parts += __shfl_xor(parts, 32, 64);
            qp = g == sub ? parts : qp;
        }
    }

    const float *M = a.means + ((int64_t)b * a.nb * a.hk + h) * a.d;
    const int64_t mstride = (int64_t)a.hk * a.d;
    float next[DP / 32][8];
    auto fetch = [&](int t0) __attribute__((always_inline)) {
        const int blk = t0 + l15;
#pragma unroll
        for (int kk = 0; kk < DP / 32; ++kk) {
            const int c = kk * 32 + g * 8;
            hd_f4 x0 = {0.f, 0.f, 0.f, 0.f}, x1 = x0;
            if (blk < most && c < a.d) {
                const float *p = M + blk * mstride + c;
                x0 = *(const hd_f4 *)p;
                x1 = *(const hd_f4 *)(p + 4);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                next[kk][j] = x0[j], next[kk][4 + j] = x1[j];
        }
    };
    float mn = 0.f;                         // largest |mean|^2 of this lane's blocks; not finite: ambiguous
    bool odd = false;
    // the 16 scores of block t0 .. t0 + 15 for query `lane`
    auto scores = [&](int t0, bool norms, float *x) __attribute__((always_inline)) {
        BtSplit m[DP / 32];
        float n2 = 0.f;
#pragma unroll
        for (int kk = 0; kk < DP / 32; ++kk) {
            m[kk] = bt_split(next[kk]);
            if (norms)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    n2 = __builtin_fmaf(next[kk][j], next[kk][j], n2);
        }
        if (norms) {
            n2 += __shfl_xor(n2, 16, 64);
            n2 += __shfl_xor(n2, 32, 64);
            odd |= !(n2 <= 3.4028235e38f);
            mn = fmaxf(mn, n2);
        }
        if (t0 + 16 < most)
            fetch(t0 + 16);
#pragma unroll
        for (int sub = 0; sub < 4; ++sub) {
            hd_f4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kk = 0; kk < DP / 32; ++kk) {
                c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(m[kk].lo, q[sub][kk].hi, c, 0, 0, 0);
                if (LOQ)
                    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(m[kk].hi, q[sub][kk].lo, c, 0, 0, 0);
                c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(m[kk].hi, q[sub][kk].hi, c, 0, 0, 0);
            }
            *(hd_f4 *)(sc + (sub * 16 + l15) * BT_STRIDE + g * 4) = c;
        }
        bt_exchange();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const hd_f4 v = *(const hd_f4 *)(sc + lane * BT_STRIDE + j * 4);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                x[j * 4 + r] = v[r];
        }
        bt_exchange();
    };

    float best[NL];                         // descending; the first NL - 1 - EXTRA - k places are held by infinities
#pragma unroll
    for (int j = 0; j < NL; ++j)
        best[j] = j < NL - 1 - EXTRA - k ? INFINITY : -INFINITY;
    const uint32_t low = IDS ? 0xFFFFFFFFu >> __clz(a.nb | 1) : 0u;     // the bits of a block's number
    const bool everything = end <= k;
    if (__any(!everything)) {
        if (most > 0)
            fetch(0);
        for (int t0 = 0; t0 < most; t0 += 16) {
            float x[16];
            scores(t0, true, x);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                float v = x[e];
                if constexpr (IDS)
                    v = __uint_as_float((__float_as_uint(v) & ~low) | (uint32_t)(t0 + e));
                v = t0 + e < end ? v : -INFINITY;
#pragma unroll
                for (int j = NL - 1; j > 0; --j)
                    best[j] = __builtin_amdgcn_fmed3f(best[j - 1], best[j], v);
                best[0] = fmaxf(best[0], v);
            }
        }
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1)
        mn = fmaxf(mn, __shfl_xor(mn, o, 64));
    // 2 eps; the heads' fp32 sums: off by (group - 1) 2^-24 sum |q_h| <= (group - 1) 2^-24 sqrt(group sum |q_h|^2)
    const float heads = (float)(a.group - 1) * 2.384185791015625e-7f * sqrtf((float)a.group * qp);
    // (a number in the score's lowest bits moves it by at most `low` 2^-23 of itself)
    constexpr float OUT = (LOQ ? 3.f : 1.f) / 262144.f, ADD = (LOQ ? 3.f : 2.f) / 8388608.f;
    const float eps2 = (2.f * (OUT + ADD * (float)a.d + (float)low / 8388608.f) * sqrtf(qn) + heads) * sqrtf(mn);
    // (squares near the smallest numbers of fp32 say nothing)
    const bool bounded = !__any(odd) && qn > 1e-30f && mn > 1e-30f && qn < 1e37f && mn < 1e37f;
    const float kth = best[NL - 2 - EXTRA], after = best[NL - 1 - EXTRA];
    const bool plain = everything || k == 0 || (bounded && kth - after > eps2 && kth < INFINITY);
    // blocks above `in` are picked, those from `near` on may be
    const float in = everything ? -INFINITY : plain ? after : after + eps2, near = plain ? INFINITY : kth - eps2;
    bool open = !plain && (!bounded || !(fabsf(kth) < INFINITY) || !(fabsf(after) < INFINITY));
    int at = 0, certain = 0;
    if constexpr (IDS) {
        // the list holds them; it holds all near ones if its end is not one of them
        open |= !plain && best[NL - 1] >= near;
#pragma unroll
        for (int j = 0; j < NL; ++j) {
            const bool sure = best[j] > in, here = best[j] < INFINITY && (sure || best[j] >= near) && !everything;
            const int id = (int)(__float_as_uint(best[j]) & low);
            if (here)
                found[at * 64 + lane] = id + (sure ? 0 : BT_NEAR);
            at += here;
            certain += here && sure;
        }
        if (everything)
            for (at = 0; at < end; ++at)
                found[at * 64 + lane] = at;
    } else if (k > 0) {
        if (most > 0)
            fetch(0);
        for (int t0 = 0; t0 < most; t0 += 16) {
            float x[16];
            scores(t0, false, x);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const bool sure = everything || x[e] > in;
                if (t0 + e < end && (sure || x[e] >= near)) {
                    if (at < places)
                        found[at * 64 + lane] = t0 + e + (sure ? 0 : BT_NEAR);
                    ++at;
                    certain += sure;
                }
            }
        }
    }
    open |= !plain && at > places;
    open &= i < lm;
    bt_exchange();                          // lanes read what others found
    for (unsigned long long left = __ballot(!plain && !open && i < lm); left; left &= left - 1) {
        const int f = __ffsll(left) - 1, all = __shfl(at, f, 64), want = k - __shfl(certain, f, 64);
        const int mine = lane < all ? found[lane * 64 + f] : 0;
        const bool unsure = (mine & BT_NEAR) != 0;
        const unsigned long long near_ones = __ballot(unsure);
        double qv[DP / 64 > 0 ? DP / 64 : 1];
#pragma unroll
        for (int c = 0; c < (DP / 64 > 0 ? DP / 64 : 1); ++c) {
            qv[c] = 0.0;
            if (c * 64 + lane < a.d)
                for (int e = 0; e < a.group; ++e)
                    qv[c] += (double)(float)Q[(i0 + f) * a.q.sr + e * a.q.sh + c * 64 + lane];
        }
        uint64_t key = 0;
        for (unsigned long long u = near_ones; u; u &= u - 1) {
            const int e = __ffsll(u) - 1;
            const float *p = M + (__shfl(mine, e, 64) & ~BT_NEAR) * mstride;
            double v = 0.0;
#pragma unroll
            for (int c = 0; c < (DP / 64 > 0 ? DP / 64 : 1); ++c)
                if (c * 64 + lane < a.d)
                    v = __builtin_fma((double)p[c * 64 + lane], qv[c], v);
#pragma unroll
            for (int o = 32; o > 0; o >>= 1)
                v += __shfl_xor(v, o, 64);
            key = lane == e ? bs_key(v) : key;
        }
        int rank = 0;
        for (unsigned long long u = near_ones; u; u &= u - 1) {
            const int e = __ffsll(u) - 1;
            const uint64_t other = __shfl((unsigned long long)key, e, 64);
            rank += other > key || (other == key && __shfl(mine, e, 64) < mine) ? 1 : 0;
        }
        const bool stays = lane < all && (!unsure || rank < want);
        const unsigned long long kept = __ballot(stays);
        if (stays)
            found[__popcll(kept & ((1ull << lane) - 1)) * 64 + f] = mine & ~BT_NEAR;
        at = lane == f ? __popcll(kept) : at;
    }
    bt_exchange();                          // and this lane's list as others left it
    at = min(at, k);                        // (open queries may hold more)
    if constexpr (IDS) {                    // ascending
        int id[NL - 1 - EXTRA];
#pragma unroll
        for (int j = 0; j < NL - 1 - EXTRA; ++j)
            id[j] = j < at ? found[j * 64 + lane] & ~BT_NEAR : 0x7FFFFFFF;
#pragma unroll
        for (int x = 0; x < NL - 1 - EXTRA; ++x)
#pragma unroll
            for (int j = x & 1; j + 1 < NL - 1 - EXTRA; j += 2) {
                const int lo = min(id[j], id[j + 1]), hi = max(id[j], id[j + 1]);
                id[j] = lo, id[j + 1] = hi;
            }
#pragma unroll
        for (int j = 0; j < NL - 1 - EXTRA; ++j)
            if (j < at)
                found[j * 64 + lane] = id[j];
    }
    if (own >= 0)
        found[at++ * 64 + lane] = own;      // behind all others: they are earlier blocks
    for (; at < a.count; ++at)
        found[at * 64 + lane] = -1;
    const unsigned long long opened = __ballot(open);
    if (lane == 0)
        a.open[w] = opened;
    bt_exchange();
    int32_t *out = a.out + (((int64_t)b * a.m + i0) * a.hk + h) * a.count;
    const int rows = min(64, a.m - i0);
    for (int e = lane; e < rows * a.count; e += 64) {
        const int r = e / a.count, j = e - r * a.count;
        out[(int64_t)r * a.hk * a.count + j] = found[j * 64 + r];
    }
}

// Parts of the blocks where there are few queries.  Up to 256 blocks one workgroup is faster than parts and the launch that joins
// them (64 channels, 80 blocks, 1 / 64 / 512 queries: 5.6 / 5.8 / 6.6 us for 8.8 / 9.3 / 11.6; 256 blocks: 6.8 / 7.1 / 8.3 for 8.8 /
// 9.4 / 12.0); beyond, parts of 128 blocks up to four workgroups a compute unit, two for up to 64 queries (2048 blocks of 128
// channels, 64 queries: 18 for 20; 256: 35 with four, 48 with two; 1000 blocks, 64: 11.5 for 15.3).
int bs_splits(int b, int m, int hk, int nb, int count)
{
    const int64_t rows = (int64_t)b * m * hk;
    if (rows <= 0 || nb <= 256)
        return 1;
    int64_t s = (rows <= 64 ? 512 : 1024) / rows;
    s = s < (nb + 127) / 128 ? s : (nb + 127) / 128;
    s = s < BS_KEEP / count ? s : BS_KEEP / count;
    return s < 1 ? 1 : (int)s;
}

// A lane per query once there are enough of them to fill the chip with waves of 64: its time hardly depends on the number of
// queries below that (64 channels, 80 blocks: 24 - 30 us), a workgroup per query costs more with each (10 us for 256 queries,
// 12 for 2048, 22 for 4096, 36 for 8192, 43 for 10000).  More blocks lengthen the lane's chain: at 500 blocks 4096 queries take
// 89 us against 45, 8192 take 90 against 81 (128 channels: 121 against 140) and 12000 take 90 against 116.
bool bs_many(int b, int m, int hk, int nb) { return m >= 16 && (int64_t)b * m * hk >= (nb <= 128 ? 4096 : 8192); }

template <typename T, int DP, bool LOQ> int bs_many_launch(const BsArgs &a, hipStream_t s)
{
    const int qtiles = (a.m - 1) / 64 + 1, k = a.count - a.causal;
    const int64_t waves = (int64_t)a.b * a.hk * qtiles;
    size_t lds;
    const int most = 4 * 64 * (BT_STRIDE + 64) * 4;             // the same in every call: another thread's does not lower it
    const dim3 grid((unsigned)((waves + 3) / 4));
    hipError_t e = hipSuccess;
#define BT_GO(NL, IDS)                                                                                                   \
    {                                                                                                                    \
        const int places = IDS ? (NL > a.count ? NL : a.count) : a.count + BT_MORE < 64 ? a.count + BT_MORE : 64;        \
        lds = (size_t)4 * 64 * (BT_STRIDE + (places > a.count ? places : a.count)) * 4;                                  \
        e = hipFuncSetAttribute((const void *)block_select_many_kernel<T, DP, NL, LOQ, IDS>,                             \
                                hipFuncAttributeMaxDynamicSharedMemorySize, most);                                       \
        if (e == hipSuccess)                                                                                             \
            hipLaunchKernelGGL((block_select_many_kernel<T, DP, NL, LOQ, IDS>), grid, dim3(BS_THREADS), lds, s, a, qtiles, waves); \
    }
    const bool ids = a.nb <= 1024;
    if (ids && k <= 4)
        BT_GO(4 + 1 + BT_EXTRA, true)
    else if (ids && k <= 8)
        BT_GO(8 + 1 + BT_EXTRA, true)
    else if (ids && k <= 16)
        BT_GO(16 + 1 + BT_EXTRA, true)
    else if (k <= 16)
        BT_GO(17, false)
    else if (k <= 32)
        BT_GO(33, false)
    else
        BT_GO(65, false)
#undef BT_GO
    if (e != hipSuccess)
        return (int)e;
    const int64_t units = waves * BO_PARTS;
    hipLaunchKernelGGL((block_select_open_kernel<T, DP>), dim3((unsigned)(units < 1024 ? units : 1024)), dim3(BS_THREADS), 0, s, a, qtiles, waves);
    return tpu3_launch_status();
}
template <typename T, bool LOQ> int bs_many_d(const BsArgs &a, hipStream_t s)
{
    return a.d <= 32 ? bs_many_launch<T, 32, LOQ>(a, s) : a.d <= 64 ? bs_many_launch<T, 64, LOQ>(a, s) : bs_many_launch<T, 128, LOQ>(a, s);
}

}  // namespace

extern "C" int tpu3_block_means(tpu3_stream_t stream, int type, int b, int n, int d, const tpu3_heads *k,
                                const int32_t *n_arr, int last, float *means)
{
    if (b < 0 || n < 0 || d <= 0 || !hd_type_ok(type) || !k || k->heads <= 0)
        return TPU3_EINVAL;
    if (d % 8 || d > 128 || (int64_t)k->heads * d > 0x7FFFFFFF)
        return TPU3_ELIMIT;
    if (b == 0 || n == 0 || last == 0)
        return TPU3_OK;
    if (!hd_rows_ok(k, type) || !means || ((uintptr_t)means & 15))
        return TPU3_EINVAL;
    const int nb = (n - 1) / BS_BLOCK + 1;
    int blocks = nb;
    if (last > 0 && (last - 1) / BS_BLOCK + 2 < blocks)
        blocks = (last - 1) / BS_BLOCK + 2;
    if ((int64_t)b * blocks >= 1 << 24)     // (2^32 threads a launch)
        return TPU3_ELIMIT;
    const hipStream_t s = (hipStream_t)stream;
    const dim3 grid((unsigned)(b * blocks));
#define BM_GO(T) hipLaunchKernelGGL(block_means_kernel<T>, grid, dim3(BS_THREADS), 0, s, n, d, nb, blocks, last, *k, n_arr, means)
    if (type == TPU3_TYPE_F32)
        BM_GO(float);
    else if (type == TPU3_TYPE_F16)
        BM_GO(_Float16);
    else
        BM_GO(__bf16);
#undef BM_GO
    return tpu3_launch_status();
}

extern "C" size_t tpu3_block_select_workspace_bytes(int b, int m, int n, int hk, int count)
{
    if (b <= 0 || m <= 0 || n <= 0 || hk <= 0 || count <= 0 || count > BS_MAX)
        return 0;
    if (bs_many(b, m, hk, (n - 1) / BS_BLOCK + 1))
        return (size_t)b * hk * (((size_t)m + 63) / 64) * 8;
    const int splits = bs_splits(b, m, hk, (n - 1) / BS_BLOCK + 1, count);
    return splits == 1 ? 0 : (size_t)b * m * hk * splits * count * 12;
}

extern "C" int tpu3_block_select(tpu3_stream_t stream, int type, int b, int m, int n, int d, const tpu3_heads *q, int hk,
                                 const float *means, const int32_t *n_arr, const int32_t *m_arr, int causal, int count,
                                 int32_t *blocks, void *workspace, size_t workspace_bytes)
{
    if (b < 0 || m < 0 || n < 0 || d <= 0 || hk <= 0 || !hd_type_ok(type) || !q || q->heads <= 0 || q->heads % hk || count <= 0)
        return TPU3_EINVAL;
    if (d % 8 || d > 128 || count > BS_MAX || (n > 0 && (n - 1) / BS_BLOCK + 1 > TPU3_ATTN_BLOCKS_MAX))
        return TPU3_ELIMIT;
    if (b == 0 || m == 0)
        return TPU3_OK;
    if (!hd_rows_ok(q, type) || !blocks || (n > 0 && (!means || ((uintptr_t)means & 15))))
        return TPU3_EINVAL;
    BsArgs a = {};
    a.q = *q, a.means = means, a.n_arr = n_arr, a.m_arr = m_arr, a.out = blocks;
    a.b = b, a.m = m, a.n = n, a.nb = n > 0 ? (n - 1) / BS_BLOCK + 1 : 0, a.hk = hk, a.group = q->heads / hk, a.d = d;
    a.count = count, a.causal = causal != 0;
    a.splits = a.nb ? bs_splits(b, m, hk, a.nb, count) : 1;
    const int64_t rows = (int64_t)b * m * hk;
    const bool many = a.nb > 0 && bs_many(b, m, hk, a.nb);
    if (many)
        a.splits = 1;
    // (2^32 threads a launch)
    const int64_t workgroups = many ? ((int64_t)b * hk * ((m - 1) / 64 + 1) + 3) / 4 : rows * a.splits;
    if (rows > 0x7FFFFFFFLL || m > 0x7FFFFFFF - 63 || workgroups >= 1 << 24)
        return TPU3_ELIMIT;
    const hipStream_t s = (hipStream_t)stream;
    if (many) {
        if (!workspace || ((uintptr_t)workspace & 7) || workspace_bytes < tpu3_block_select_workspace_bytes(b, m, n, hk, count))
            return TPU3_EINVAL;
        a.open = (uint64_t *)workspace;
        // (bf16 queries of one head are their own first term)
        return type == TPU3_TYPE_F32   ? bs_many_d<float, true>(a, s)
               : type == TPU3_TYPE_F16 ? bs_many_d<_Float16, true>(a, s)
               : a.group == 1          ? bs_many_d<__bf16, false>(a, s)
                                       : bs_many_d<__bf16, true>(a, s);
    }
    if (a.splits > 1) {
        if (!workspace || ((uintptr_t)workspace & 7) || workspace_bytes < (size_t)rows * a.splits * count * 12)
            return TPU3_EINVAL;
        a.ws_key = (uint64_t *)workspace;
        a.ws_id = (int32_t *)(a.ws_key + rows * a.splits * count);
    }
    const dim3 grid((unsigned)(rows * a.splits));
#define BS_GO(T)                                                                                                    \
    {                                                                                                               \
        if (d <= 32)                                                                                                \
            hipLaunchKernelGGL((block_select_kernel<T, 32>), grid, dim3(BS_THREADS), 0, s, a);                      \
        else if (d <= 64)                                                                                           \
            hipLaunchKernelGGL((block_select_kernel<T, 64>), grid, dim3(BS_THREADS), 0, s, a);                      \
        else                                                                                                        \
            hipLaunchKernelGGL((block_select_kernel<T, 128>), grid, dim3(BS_THREADS), 0, s, a);                     \
    }
    if (type == TPU3_TYPE_F32)
        BS_GO(float)
    else if (type == TPU3_TYPE_F16)
        BS_GO(_Float16)
    else
        BS_GO(__bf16)
#undef BS_GO
    if (a.splits > 1)
        hipLaunchKernelGGL(block_select_join_kernel, dim3((unsigned)rows), dim3(BS_THREADS), 0, s, a);
    return tpu3_launch_status();
}
