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
    // all blocks, or from the block of the first of the `last` newest rows on
    const int blk = j + (last >= 0 ? max(0, live - last) / BS_BLOCK : 0);
    if (blk >= nb)
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
    double *ws_score;                       // (b, hk, m, splits, count)
    int32_t *ws_id;
    int32_t *todo, *todo_rows;              // queries that the approximate scores leave open: their number, their rows
    int b, m, n, nb, hk, group, d, count, causal, splits;
};

constexpr int BS_KEEP = 1024;               // candidates in LDS at a time
constexpr int BS_MAX = TPU3_BLOCK_COUNT_MAX;

struct BsShared {
    double q[128];
    double score[BS_KEEP];
    int id[BS_KEEP];
    double wave_score[4 * BS_MAX];
    int wave_id[4 * BS_MAX];
};

__device__ __forceinline__ bool bs_better(double a, int ia, double b, int ib) { return a > b || (a == b && ia < ib); }

// The `count` best of the n candidates in s.score / s.id, best first, into their first places; the rest of these places is
// filled with (-inf, INT_MAX).  Every wave extracts the best of a quarter one by one; their 4 * count meet by rank.
__device__ void bs_best(BsShared &s, int n, int count)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double v[4];
    int id[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int e = wave * 256 + j * 64 + lane;
        v[j] = e < n ? s.score[e] : -INFINITY;
        id[j] = e < n ? s.id[e] : 0x7FFFFFFF;
    }
    for (int r = 0; r < count; ++r) {
        double bv = v[0];
        int bi = id[0];
#pragma unroll
        for (int j = 1; j < 4; ++j)
            if (bs_better(v[j], id[j], bv, bi))
                bv = v[j], bi = id[j];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const double ov = __shfl_xor(bv, o, 64);
            const int oi = __shfl_xor(bi, o, 64);
            if (bs_better(ov, oi, bv, bi))
                bv = ov, bi = oi;
        }
        if (lane == 0)
            s.wave_score[wave * count + r] = bv, s.wave_id[wave * count + r] = bi;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (id[j] == bi)
                v[j] = -INFINITY, id[j] = 0x7FFFFFFF;
    }
    __syncthreads();
    const int c = threadIdx.x;              // 4 * count <= 256 candidates, one a thread
    if (c < 4 * count) {
        const double cv = s.wave_score[c];
        const int ci = s.wave_id[c];
        int rank = 0;
        for (int o = 0; o < 4 * count; ++o) {
            const double ov = s.wave_score[o];
            const int oi = s.wave_id[o];
            rank += bs_better(ov, oi, cv, ci) || (ov == cv && oi == ci && o < c) ? 1 : 0;
        }
        if (rank < count)
            s.score[rank] = cv, s.id[rank] = ci;
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
template <typename T> __device__ void block_select_row(const BsArgs &a, BsShared &s, int64_t row, int z)
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
            for (int g = 0; g < a.group; ++g)
                v += (double)(float)Q[g * a.q.sh + c];
        s.q[c] = v;
    }
    __syncthreads();
    const int slot = threadIdx.x >> 3, part = threadIdx.x & 7;
    int kept = 0;                                               // candidates in LDS
    for (int c0 = z0; c0 < z1 || c0 == z0;) {
        const int take = min(z1 - c0, BS_KEEP - kept);
        for (int t0 = 0; t0 < take; t0 += BS_THREADS / 8) {
            const int t = t0 + slot, blk = c0 + t;
            double v = 0.0;
            if (t < take) {
                const float *M = a.means + (((int64_t)b * a.nb + blk) * a.hk + h) * a.d;
                for (int c = part * 4; c < a.d; c += 32) {
                    const hd_f4 x = *(const hd_f4 *)(M + c);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        v = __builtin_fma((double)x[j], s.q[c + j], v);
                }
            }
#pragma unroll
            for (int o = 4; o > 0; o >>= 1)
                v += __shfl_xor(v, o, 64);
            if (t < take && part == 0) {
                v = v == v ? v : -INFINITY;                     // not a number: behind every number
                s.score[kept + t] = blk == own ? INFINITY : v;
                s.id[kept + t] = blk;
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
        a.ws_score[at] = s.score[threadIdx.x];
        a.ws_id[at] = s.id[threadIdx.x];
    }
}

template <typename T>
__global__ __launch_bounds__(BS_THREADS) void block_select_kernel(BsArgs a)
{
    __shared__ BsShared s;
    if (a.todo) {                           // the rows of a list
        const int all = *a.todo;
        for (int r = blockIdx.x; r < all; r += gridDim.x) {
            block_select_row<T>(a, s, a.todo_rows[r], 0);
            __syncthreads();
        }
        return;
    }
    block_select_row<T>(a, s, blockIdx.x / a.splits, (int)(blockIdx.x % a.splits));
}

__global__ __launch_bounds__(BS_THREADS) void block_select_join_kernel(BsArgs a)
{
    __shared__ BsShared s;
    const int64_t row = blockIdx.x;
    const int i = (int)(row % a.m);
    const int bh = (int)(row / a.m), h = bh % a.hk, b = bh / a.hk;
    const int all = a.splits * a.count;                         // <= BS_KEEP by the host's choice of splits
    for (int t = threadIdx.x; t < all; t += BS_THREADS) {
        s.score[t] = a.ws_score[row * all + t];
        s.id[t] = a.ws_id[row * all + t];
    }
    __syncthreads();
    bs_best(s, all, a.count);
    bs_emit(s, a.count, a.out + (((int64_t)b * a.m + i) * a.hk + h) * a.count);
}

// ---- selection for many queries ------------------------------------------------------------------------------------------
// A lane per query, 64 queries of one key head a wave.  The scores come from the matrix cores, approximately, with a bound:
// queries and means as two bf16 terms each (hi + lo, |x - hi - lo| <= 2^-18 |x|), three of the four partial products, fp32
// sums: off by at most  eps = 2^-13 |q| max_b |mean_b|  (3 * 2^-18 for the terms left out, 3 d * 2^-24 = 2^-15.4 at d = 128
// for the sums, doubled for sums that cut off instead of rounding).  Pass 1 keeps the k + 1 largest scores of every query, a
// chain of v_med3 (one instruction an entry).  Where the k-th is more than 2 eps above the next, the order of the exact
// scores around that place is known, and pass 2, which forms the same scores again, lists the blocks above it in ascending
// order.  The other queries (near ties, equal rows, values that are not finite; a few in a thousand) are put on a list
// for block_select_kernel's exact scores.
constexpr int BT_STRIDE = 20;               // floats between two queries' 16 scores in LDS

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

template <typename T, int DP, int NL, bool LOQ>
__global__ __launch_bounds__(BS_THREADS) void block_select_many_kernel(BsArgs a, int qtiles, int64_t waves)
{
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, g = lane >> 4;
    float *sc = (float *)smem + wave * (64 * BT_STRIDE);
    int *found = (int *)((float *)smem + 4 * 64 * BT_STRIDE) + wave * 64 * a.count;          // (count, 64)
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
    float qn = 0.f;                         // |q|^2 of query `lane`
    const T *Q = (const T *)a.q.data + b * a.q.sb + (int64_t)h * a.group * a.q.sh;
#pragma unroll
    for (int sub = 0; sub < 4; ++sub) {
        const int r = i0 + sub * 16 + l15;
        float n2 = 0.f;
#pragma unroll
        for (int kk = 0; kk < DP / 32; ++kk) {
            const int c = kk * 32 + g * 8;
            float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (r < lm && c < a.d)
                for (int e = 0; e < a.group; ++e) {
                    float y[8];
                    hd_load8(Q + r * a.q.sr + e * a.q.sh + c, y);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        x[j] += y[j];
                }
#pragma unroll
            for (int j = 0; j < 8; ++j)
                n2 = __builtin_fmaf(x[j], x[j], n2);
            q[sub][kk] = bt_split(x);
        }
        n2 += __shfl_xor(n2, 16, 64);
        n2 += __shfl_xor(n2, 32, 64);
        qn = g == sub ? n2 : qn;            // lane sub*16 + l15
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
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();    // (one wave: its LDS accesses complete in order)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const hd_f4 v = *(const hd_f4 *)(sc + lane * BT_STRIDE + j * 4);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                x[j * 4 + r] = v[r];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };

    float best[NL];                         // descending; the first NL - 1 - k places are held by infinities
#pragma unroll
    for (int j = 0; j < NL; ++j)
        best[j] = j < NL - 1 - k ? INFINITY : -INFINITY;
    const bool everything = end <= k;
    if (__any(!everything)) {
        if (most > 0)
            fetch(0);
        for (int t0 = 0; t0 < most; t0 += 16) {
            float x[16];
            scores(t0, true, x);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float v = t0 + e < end ? x[e] : -INFINITY;
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
    const float eps = 1.220703125e-4f * sqrtf(qn) * sqrtf(mn);
    const bool any_odd = __any(odd);
    const bool sure = everything || k == 0 || (!any_odd && best[NL - 2] - best[NL - 1] > 2.f * eps && best[NL - 2] < INFINITY);
    const float above = everything ? -INFINITY : best[NL - 1];
    int at = 0;
    if (k > 0) {
        if (most > 0)
            fetch(0);
        for (int t0 = 0; t0 < most; t0 += 16) {
            float x[16];
            scores(t0, false, x);
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (t0 + e < end && (everything || x[e] > above) && at < k)
                    found[at++ * 64 + lane] = t0 + e;
        }
    }
    if (own >= 0)
        found[at++ * 64 + lane] = own;      // behind all others: they are earlier blocks
    for (; at < a.count; ++at)
        found[at * 64 + lane] = -1;
    if (i < lm && !sure) {
        const int slot = atomicAdd(a.todo, 1);
        a.todo_rows[slot] = (int)((int64_t)bh * a.m + i);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    int32_t *out = a.out + (((int64_t)b * a.m + i0) * a.hk + h) * a.count;
    const int rows = min(64, a.m - i0);
    for (int e = lane; e < rows * a.count; e += 64) {
        const int r = e / a.count, j = e - r * a.count;
        out[(int64_t)r * a.hk * a.count + j] = found[j * 64 + r];
    }
}

// Parts of the blocks: enough workgroups for the chip when there are few queries (a part holds 64 blocks at least).
int bs_splits(int b, int m, int hk, int nb, int count)
{
    const int64_t rows = (int64_t)b * m * hk;
    if (rows <= 0)
        return 1;
    int64_t s = 1024 / rows;
    s = s < (nb + 63) / 64 ? s : (nb + 63) / 64;
    s = s < BS_KEEP / count ? s : BS_KEEP / count;
    return s < 1 ? 1 : (int)s;
}

// A lane per query once there are enough of them.
bool bs_many(int b, int m, int hk) { return m >= 16 && (int64_t)b * m * hk >= 512; }

template <typename T, int DP, bool LOQ> int bs_many_launch(const BsArgs &a, hipStream_t s)
{
    const int qtiles = (a.m + 63) / 64, k = a.count - a.causal;
    const int64_t waves = (int64_t)a.b * a.hk * qtiles;
    const size_t lds = (size_t)4 * 64 * (BT_STRIDE + a.count) * 4;
    const dim3 grid((unsigned)((waves + 3) / 4));
    hipError_t e = hipSuccess;
#define BT_GO(NL)                                                                                                        \
    {                                                                                                                    \
        e = hipFuncSetAttribute((const void *)block_select_many_kernel<T, DP, NL, LOQ>,                                  \
                                hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);                                   \
        if (e == hipSuccess)                                                                                             \
            hipLaunchKernelGGL((block_select_many_kernel<T, DP, NL, LOQ>), grid, dim3(BS_THREADS), lds, s, a, qtiles, waves); \
    }
    if (k < 5)
        BT_GO(5)
    else if (k < 9)
        BT_GO(9)
    else if (k < 17)
        BT_GO(17)
    else if (k < 33)
        BT_GO(33)
    else
        BT_GO(65)
#undef BT_GO
    return e == hipSuccess ? tpu3_launch_status() : (int)e;
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
    if (d % 8 || d > 128)
        return TPU3_ELIMIT;
    if (b == 0 || n == 0 || last == 0)
        return TPU3_OK;
    if (!hd_rows_ok(k, type) || !means || ((uintptr_t)means & 15))
        return TPU3_EINVAL;
    const int nb = (n - 1) / BS_BLOCK + 1;
    int blocks = nb;
    if (last > 0 && (last - 1) / BS_BLOCK + 2 < blocks)
        blocks = (last - 1) / BS_BLOCK + 2;
    if ((int64_t)b * blocks > 0x7FFFFFFFLL)
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
    if (bs_many(b, m, hk))
        return ((size_t)b * m * hk + 2) * 4;
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
    const bool many = a.nb > 0 && bs_many(b, m, hk);
    if (many)
        a.splits = 1;
    if (rows * a.splits > 0x7FFFFFFFLL)
        return TPU3_ELIMIT;
    const hipStream_t s = (hipStream_t)stream;
    if (many) {
        if (!workspace || ((uintptr_t)workspace & 7) || workspace_bytes < ((size_t)rows + 2) * 4)
            return TPU3_EINVAL;
        a.todo = (int32_t *)workspace, a.todo_rows = a.todo + 2;
        const hipError_t e = tpu3_fill_u32(a.todo, 0, 2, s);
        if (e != hipSuccess)
            return (int)e;
        const bool bf16 = type == TPU3_TYPE_BF16;
        const int rc = type == TPU3_TYPE_F32 ? bs_many_d<float, true>(a, s)
                       : !bf16               ? bs_many_d<_Float16, true>(a, s)
                       : a.group == 1        ? bs_many_d<__bf16, false>(a, s)
                                             : bs_many_d<__bf16, true>(a, s);
        if (rc)
            return rc;
    }
    if (a.splits > 1) {
        if (!workspace || ((uintptr_t)workspace & 7) || workspace_bytes < (size_t)rows * a.splits * count * 12)
            return TPU3_EINVAL;
        a.ws_score = (double *)workspace;
        a.ws_id = (int32_t *)(a.ws_score + rows * a.splits * count);
    }
    const dim3 grid((unsigned)(many ? (rows < 1024 ? rows : 1024) : rows * a.splits));
#define BS_GO(T) hipLaunchKernelGGL(block_select_kernel<T>, grid, dim3(BS_THREADS), 0, s, a)
    if (type == TPU3_TYPE_F32)
        BS_GO(float);
    else if (type == TPU3_TYPE_F16)
        BS_GO(_Float16);
    else
        BS_GO(__bf16);
#undef BS_GO
    if (a.splits > 1)
        hipLaunchKernelGGL(block_select_join_kernel, dim3((unsigned)rows), dim3(BS_THREADS), 0, s, a);
    return tpu3_launch_status();
}
