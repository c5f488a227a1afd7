// norm_rotate.hip -- per-head RMS norm of queries and keys with the position rotation in the same pass, and its gradient.
//
//   r = 1 / sqrt(mean_c x_c^2 + eps),  u = x r,  y = u w,  then every pair (one, two) of the rotated channels turns by the
//   angle position[axis] * freq[axis][f]:  (y_one c - y_two s,  y_one s + y_two c);  channels behind the pairs pass.
//   Backward, with h = the gradient turned back by the same angle:
//   dx = r (h w - u mean_c(h w u)),  dw = sum over rows of h u.
//
// Bound by memory: a row is read once and written once (backward: read twice, written once), ~20 flops a channel.  A lane
// holds eight consecutive channels (one 16-byte access for the 16-bit types); 4 .. 32 lanes hold a row, so that the sums
// of a row are a few lane exchanges.  The turns are shared by all heads of a token: a workgroup takes a few tokens,
// computes their cosines and sines once into LDS and then runs over the tokens' rows.  Angles are formed and reduced in
// 64 bits (a position of 1e5 times a frequency of 1 leaves 7 of fp32's 24 bits for the fraction of a turn), the sine and
// cosine of the fraction in 32.  Both pair orders use one expression, z[c] = y[c] C[c] + y[partner(c)] S[c], with the sign
// folded into S and C = 1, S = 0 behind the pairs.  In the half-split order the partner sits in another lane: the normed row
// goes through LDS with its first half stored a second time behind the second, so that the partner of channel c is always
// channel c + P (P pairs; lane exchanges where P is a multiple of eight).
// The next row is requested before the current one is worked on (a wave otherwise has 1 KB in flight, and the chip 7 MB).
// Results are stored past the caches: this kernel alone is faster for it, a program hardly, since who reads the results next
// finds fewer of them cached.  us with ordinary stores / with these, 8 + 8 heads of 64 channels, bf16: a cloud of 80000 points,
// rotation 101 / 76, with attention behind it 387 / 386, forward and backward 1953 / 1941; 16 clouds of 5000 100 / 73, 352 / 357,
// 1290 / 1312; 8 clouds 41 / 40, 164 / 162, 668 / 679; 2 clouds 17 / 15, 55 / 54, 226 / 225.
#include "heads.h"

namespace {

constexpr int NR_THREADS = 256;
constexpr size_t NR_LDS = 160 * 1024;
constexpr int NR_MAX_WG = 1024;             // backward: persistent workgroups, one partial weight gradient each

struct NrArgs {
    tpu3_heads x[2];                        // queries, keys (heads 0: none)
    tpu3_heads g[2];                        // backward: gradients of the outputs
    const void *w[2];
    int w_head[2];                          // channels between two heads' weights (0: one set for all heads)
    void *out[2];                           // contiguous (b, n, heads, d)
    float *part;                            // backward: (workgroups, rows of weights, d)
    int want_w[2];
    const void *pos, *freq;
    int64_t pos_sb, pos_sn, pos_sa;
    int64_t tokens;
    int n, d, axes, pairs, total_pairs, w_type, pos_type, freq_type, interleaved, tok;
    float eps, inv_d;
};

__device__ __forceinline__ void nr_weights(const void *w, int type, int i, float *y)
{
    if (!w) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            y[j] = 1.f;
    } else if (type == TPU3_TYPE_F32) {
        hd_load8((const float *)w + i, y);
    } else if (type == TPU3_TYPE_F16) {
        hd_load8((const _Float16 *)w + i, y);
    } else {
        hd_load8((const __bf16 *)w + i, y);
    }
}
__device__ __forceinline__ double nr_position(const void *p, int type, int64_t i)
{
    if (type == TPU3_POS_F32)
        return (double)((const float *)p)[i];
    if (type == TPU3_POS_F64)
        return ((const double *)p)[i];
    if (type == TPU3_POS_I32)
        return (double)((const int32_t *)p)[i];
    return (double)((const int64_t *)p)[i];
}

// C and S of the workgroup's tokens: cs[(t * 2 + which) * d + c]
__device__ __forceinline__ void nr_turns(const NrArgs &a, int64_t t0, int count, float sign, float *cs)
{
    const int P = a.total_pairs, rest = a.d - 2 * P;
    for (int i = threadIdx.x; i < count * P; i += NR_THREADS) {
        const int t = i / P, p = i - t * P, ax = p / a.pairs;
        const int64_t tok = t0 + t, e = tok / a.n, r = tok - e * a.n;
        const double pos = nr_position(a.pos, a.pos_type, e * a.pos_sb + r * a.pos_sn + ax * a.pos_sa);
        const double f = a.freq_type == TPU3_POS_F64 ? ((const double *)a.freq)[p] : (double)((const float *)a.freq)[p];
        double turn = pos * f * 0.15915494309189533577;         // 1 / (2 pi)
        turn -= rint(turn);
        float s, c;
        sincospif(2.f * (float)turn, &s, &c);
        // what the rounding of the turn took, to first order: an angle of up to 2 pi 2^-26 (fp32 outputs off by 7.8e-8 without it,
        // 7.0e-8 with it; the plain form 6.5e-8)
        const float more = 6.2831853f * (float)(turn - (double)(float)turn), s0 = s;
        s = __builtin_fmaf(c, more, s);
        c = __builtin_fmaf(-s0, more, c);
        const int one = a.interleaved ? 2 * p : p, two = a.interleaved ? 2 * p + 1 : p + P;
        float *C = cs + t * 2 * a.d, *S = C + a.d;
        C[one] = C[two] = c;
        S[one] = -sign * s;
        S[two] = sign * s;
    }
    for (int i = threadIdx.x; i < count * rest; i += NR_THREADS) {
        const int t = i / rest, c = 2 * P + (i - t * rest);
        cs[t * 2 * a.d + c] = 1.f;
        cs[(t * 2 + 1) * a.d + c] = 0.f;
    }
}

template <int LPR> __device__ __forceinline__ float nr_row_sum(float v)
{
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1)
        v += __shfl_xor(v, o, 64);
    return v;
}

// Exchange rows, for halves whose length is no multiple of eight: channel c of a row sits at (c % 8) * slots + c / 8, so that
// the lanes of a row, which hold channels 8 l .. 8 l + 7, meet different banks whatever the shift is.  The rows of a wave, 8 *
// slots apart, may still share theirs (64 channels, 30 pairs: 112 words, so the rows four apart do).  Lanes write whole
// groups of eight: what lies behind the second half is written over by the copy of the first, which is written after it, and
// what a channel behind the pairs reads is not used.
__host__ __device__ __forceinline__ int nr_slots(int d, int pairs) { return (d + pairs + 15) / 8 + 1; }
__host__ __device__ __forceinline__ bool nr_exchanges(int pairs, int interleaved) { return !interleaved && pairs % 8 != 0; }

// eight channels from c0 on turned; `row` is this row's exchange slice.  Whole rows run it (LPR lanes each).
template <int LPR> __device__ __forceinline__ void nr_turn(const NrArgs &a, const float *cs, float *row, int c0, bool live, float *y)
{
    const int P = a.total_pairs;
    float o[8];
    if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            o[i] = y[i ^ 1];
    } else if (P % 8 == 0) {                // the partner is a whole number of lanes away
        const int l = c0 >> 3, shift = P >> 3, from = l < shift ? l + shift : l < 2 * shift ? l - shift : l;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            o[i] = __shfl(y[i], from, LPR);
    } else {
        const int slots = nr_slots(a.d, P);
        if (live)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                row[i * slots + (c0 >> 3)] = y[i];
        if (c0 < P)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                row[((2 * P + i) & 7) * slots + ((2 * P + c0 + i) >> 3)] = y[i];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();    // the row's lanes are in one wave, whose LDS accesses complete in order
        if (live)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = row[((P + i) & 7) * slots + ((P + c0 + i) >> 3)];
                o[i] = c0 + i < 2 * P ? x : 0.f;
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    if (!live)
        return;
    const hd_f4 c_0 = *(const hd_f4 *)(cs + c0), c_1 = *(const hd_f4 *)(cs + c0 + 4);
    const hd_f4 s_0 = *(const hd_f4 *)(cs + a.d + c0), s_1 = *(const hd_f4 *)(cs + a.d + c0 + 4);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        y[i] = __builtin_fmaf(o[i], i < 4 ? s_0[i & 3] : s_1[i & 3], y[i] * (i < 4 ? c_0[i & 3] : c_1[i & 3]));
}

// where the tokens' rows start in the (strided) inputs: at[t] of x[0], x[1], g[0], g[1] for n of them
__device__ __forceinline__ void nr_places(const NrArgs &a, int64_t t0, int count, int n, int64_t *at)
{
    for (int i = threadIdx.x; i < count * n; i += NR_THREADS) {
        const int which = i / count, t = i - which * count;
        const int64_t tok = t0 + t, e = tok / a.n, r = tok - e * a.n;
        const tpu3_heads &x = which < 2 ? a.x[which] : a.g[which - 2];
        at[which * a.tok + t] = e * x.sb + r * x.sr;
    }
}

template <typename T, int LPR>
__global__ __launch_bounds__(NR_THREADS) void norm_rotate_kernel(NrArgs a)
{
    extern __shared__ __attribute__((aligned(16))) char smem[];
    constexpr int GROUPS = NR_THREADS / LPR;
    typedef typename hd_vec<T>::v8 V8;
    const int len = nr_exchanges(a.total_pairs, a.interleaved) ? 8 * nr_slots(a.d, a.total_pairs) : 0;
    int64_t *at = (int64_t *)smem;                              // (2, tok) places of the tokens' rows
    float *cs = (float *)(at + 2 * a.tok), *ex = cs + a.tok * 2 * a.d;      // (tok, 2, d) turns, (GROUPS, len) exchange rows
    const int64_t t0 = (int64_t)blockIdx.x * a.tok;
    const int count = (int)min((int64_t)a.tok, a.tokens - t0);
    const int grp = threadIdx.x / LPR, c0 = (threadIdx.x % LPR) * 8;
    const bool live = c0 < a.d;
    const int cr = live ? c0 : 0;           // (idle lanes of a row work on channel 0's addresses and write nothing)
    nr_places(a, t0, count, 2, at);
    nr_turns(a, t0, count, 1.f, cs);
    __syncthreads();
    const int hq = a.x[0].heads, hk = a.x[1].heads, rows = count * (hq + hk);
    const float iq = 1.f / (float)hq, ik = hk ? 1.f / (float)hk : 0.f;
    const T *X0 = (const T *)a.x[0].data + cr, *X1 = (const T *)a.x[1].data + cr;
    T *Y0 = (T *)a.out[0] + t0 * hq * a.d + c0, *Y1 = (T *)a.out[1] + t0 * hk * a.d + c0;
    // row r of the tile: queries first, token by token (r < 2^16, heads <= 1024: the rounded quotient is exact)
    auto place = [&](int r, int &side, int &t, int &h) __attribute__((always_inline)) {
        side = r >= count * hq;
        r -= side ? count * hq : 0;
        t = (int)(((float)r + 0.5f) * (side ? ik : iq));
        h = r - t * (side ? hk : hq);
    };
    auto load = [&](int r, V8 &v) __attribute__((always_inline)) {
        int side, t, h;
        place(min(r, rows - 1), side, t, h);
        v = *(const V8 *)((side ? X1 : X0) + at[side * a.tok + t] + h * (side ? a.x[1].sh : a.x[0].sh));
    };
    V8 cur, next;
    load(grp, cur);
    for (int r = grp; r < rows; r += GROUPS) {
        load(r + GROUPS, next);
        int side, t, h;
        place(r, side, t, h);
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            y[j] = live ? (float)cur[j] : 0.f;
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            ss = __builtin_fmaf(y[j], y[j], ss);
        const float inv = 1.f / sqrtf(__builtin_fmaf(nr_row_sum<LPR>(ss), a.inv_d, a.eps));
        float w[8];
        nr_weights(a.w[side], a.w_type, h * a.w_head[side] + cr, w);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            y[j] = y[j] * inv * w[j];
        nr_turn<LPR>(a, cs + t * 2 * a.d, ex + grp * len, c0, live, y);
        if (live)
            hd_stream8((side ? Y1 : Y0) + (t * (side ? hk : hq) + h) * a.d, y);
        cur = next;
    }
}

// The weight gradients: a lane adds up h u of its eight channels over the rows that its wave takes.  One set of weights for
// all heads: in registers over the whole kernel.  A set per head: a wave takes whole (head, token part) units, adds its
// lanes up after each and keeps the unit's row in LDS.  Either way a workgroup leaves one partial sum per weight, in an
// order that the sizes alone decide; norm_rotate_wsum_kernel adds the workgroups' in 64 bits.
template <typename T, int LPR>
__global__ __launch_bounds__(NR_THREADS) void norm_rotate_bwd_kernel(NrArgs a, int split)
{
    extern __shared__ __attribute__((aligned(16))) char smem[];
    constexpr int GROUPS = NR_THREADS / LPR, PER = 64 / LPR;
    typedef typename hd_vec<T>::v8 V8;
    const int heads_all = a.x[0].heads + a.x[1].heads;
    const int len = nr_exchanges(a.total_pairs, a.interleaved) ? 8 * nr_slots(a.d, a.total_pairs) : 0;
    int64_t *at = (int64_t *)smem;                              // (4, tok) places of the tokens' rows
    float *cs = (float *)(at + 4 * a.tok), *acc = cs + a.tok * 2 * a.d;     // (tok, 2, d) turns; (units, d) per-head sums
    const bool per_head = (a.w[0] && a.w_head[0]) || (a.w[1] && a.w_head[1]);
    const bool want = a.want_w[0] || a.want_w[1];
    const int units = heads_all * split;
    float *ex = acc + (want ? (per_head ? units : 8) * a.d : 0);            // (GROUPS, len) exchange rows
    const int grp = threadIdx.x / LPR, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c0 = (threadIdx.x % LPR) * 8;
    const bool live = c0 < a.d;
    const int cr = live ? c0 : 0;
    const int part_tok = (a.tok + split - 1) / split;
    float ws[2][8] = {};
    if (want && per_head)
        for (int i = threadIdx.x; i < units * a.d; i += NR_THREADS)
            acc[i] = 0.f;
    for (int64_t t0 = (int64_t)blockIdx.x * a.tok; t0 < a.tokens; t0 += (int64_t)gridDim.x * a.tok) {
        const int count = (int)min((int64_t)a.tok, a.tokens - t0);
        __syncthreads();
        nr_places(a, t0, count, 4, at);
        nr_turns(a, t0, count, -1.f, cs);
        __syncthreads();
        for (int u = wave; u < units; u += 4) {
            const int hu = u / split, s = u - hu * split;
            const int side = hu < a.x[0].heads ? 0 : 1, h = side ? hu - a.x[0].heads : hu, heads = a.x[side].heads;
            const T *X = (const T *)a.x[side].data + h * a.x[side].sh + cr;
            const T *G = (const T *)a.g[side].data + h * a.g[side].sh + cr;
            const int64_t *xa = at + side * a.tok, *ga = at + (2 + side) * a.tok;
            T *Y = (T *)a.out[side] + (t0 * heads + h) * a.d + c0;
            const int last = min(count, (s + 1) * part_tok);
            float w[8], wg[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            nr_weights(a.w[side], a.w_type, h * a.w_head[side] + cr, w);
            V8 xc = {}, gc = {}, xn = {}, gn = {};
            auto load = [&](int t, V8 &x, V8 &g) __attribute__((always_inline)) {
                t = min(t, last - 1);
                x = *(const V8 *)(X + xa[t]);
                g = *(const V8 *)(G + ga[t]);
            };
            const int tl = lane / LPR;
            if (s * part_tok >= last)
                continue;
            load(s * part_tok + tl, xc, gc);
            // (whole waves run the loop: the lanes of a row exchange values inside)
            for (int tb = s * part_tok; tb < last; tb += PER) {
                const int t = tb + tl, tc = min(t, last - 1);
                const bool row = t < last && live;
                load(t + PER, xn, gn);
                float x[8], g[8];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    x[j] = row ? (float)xc[j] : 0.f, g[j] = row ? (float)gc[j] : 0.f;
                nr_turn<LPR>(a, cs + tc * 2 * a.d, ex + grp * len, c0, live, g);
                float ss = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    ss = __builtin_fmaf(x[j], x[j], ss);
                const float inv = 1.f / sqrtf(__builtin_fmaf(nr_row_sum<LPR>(ss), a.inv_d, a.eps));
                float dot = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    x[j] *= inv;
                    wg[j] = row ? __builtin_fmaf(g[j], x[j], wg[j]) : wg[j];
                    g[j] *= w[j];
                    dot = __builtin_fmaf(g[j], x[j], dot);
                }
                dot = nr_row_sum<LPR>(dot) * a.inv_d;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    g[j] = inv * __builtin_fmaf(-x[j], dot, g[j]);
                if (row)
                    hd_stream8(Y + t * heads * a.d, g);
                xc = xn, gc = gn;
            }
            if (!want)
                continue;
            if (per_head) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
#pragma unroll
                    for (int o = LPR; o < 64; o <<= 1)
                        wg[j] += __shfl_xor(wg[j], o, 64);
                }
                if (lane < LPR && live)
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        acc[u * a.d + c0 + j] += wg[j];
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    ws[0][j] += side ? 0.f : wg[j], ws[1][j] += side ? wg[j] : 0.f;
            }
        }
    }
    if (!want)
        return;
    if (!per_head) {
#pragma unroll
        for (int side = 0; side < 2; ++side)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float v = ws[side][j];
#pragma unroll
                for (int o = LPR; o < 64; o <<= 1)
                    v += __shfl_xor(v, o, 64);
                if (lane < LPR && live)
                    acc[(side * 4 + wave) * a.d + c0 + j] = v;
            }
    }
    __syncthreads();
    const int rows = per_head ? heads_all : 2, terms = per_head ? split : 4;
    for (int i = threadIdx.x; i < rows * a.d; i += NR_THREADS) {
        const int r = i / a.d, c = i - r * a.d;
        float v = 0.f;
        for (int s = 0; s < terms; ++s)
            v += acc[(r * terms + s) * a.d + c];
        a.part[(int64_t)blockIdx.x * rows * a.d + i] = v;
    }
}

// Sums over the workgroups' partial sums of every column, in 64 bits and in a fixed order: the first nq columns to out0, the
// others to out1 (either may be absent).  Bound by latency: a thread has eight loads in flight (13 us a set, one set at a time,
// with one).
constexpr int NW_COLS = 16, NW_PARTS = 64;
__global__ __launch_bounds__(NW_COLS * NW_PARTS) void norm_rotate_wsum_kernel(int wgs, int cols, int nq, int w_type, const float *__restrict__ part,
                                                                               void *__restrict__ out0, void *__restrict__ out1)
{
    __shared__ double s[NW_PARTS][NW_COLS + 1];
    const int c = threadIdx.x % NW_COLS, g = threadIdx.x / NW_COLS, i = blockIdx.x * NW_COLS + c;
    double v = 0.0;
    if (i < cols)
#pragma unroll 8
        for (int r = g; r < wgs; r += NW_PARTS)
            v += (double)part[(int64_t)r * cols + i];
    s[g][c] = v;
    __syncthreads();
    if (g == 0 && i < cols) {
        v = 0.0;
#pragma unroll 8
        for (int r = 0; r < NW_PARTS; ++r)
            v += s[r][c];
        void *out = i < nq ? out0 : out1;
        const int at = i < nq ? i : i - nq;
        if (!out)
            return;
        if (w_type == TPU3_TYPE_F32)
            ((float *)out)[at] = (float)v;
        else if (w_type == TPU3_TYPE_F16)
            ((_Float16 *)out)[at] = (_Float16)(float)v;
        else
            ((__bf16 *)out)[at] = (__bf16)(float)v;
    }
}

struct NrPlan {
    int lpr, tok, split, wgs;
    size_t lds;
};

// Tokens of a workgroup: enough rows to fill its 256 threads, few enough that the chip's 256 compute units all get some.
NrPlan nr_plan(int64_t tokens, int heads, int d, int pairs, int interleaved, bool bwd, bool per_head, bool want)
{
    NrPlan p;
    p.lpr = d <= 32 ? 4 : d <= 64 ? 8 : d <= 128 ? 16 : 32;
    p.tok = bwd ? 64 : 16;
    while (p.tok > 1 && (tokens + p.tok - 1) / p.tok < 1024)
        p.tok >>= 1;
    while (p.tok > 1 && (size_t)p.tok * d * 8 > 32768)
        p.tok >>= 1;
    const int64_t tiles = (tokens + p.tok - 1) / p.tok;
    p.split = bwd && heads % 4 ? (p.tok >= 4 ? 4 : 1) : 1;
    p.wgs = bwd ? (int)(tiles < NR_MAX_WG ? tiles : NR_MAX_WG) : 0;
    p.lds = (size_t)p.tok * (d * 8 + (bwd ? 32 : 16));
    if (nr_exchanges(pairs, interleaved))
        p.lds += (size_t)(NR_THREADS / p.lpr) * 8 * nr_slots(d, pairs) * 4;
    if (bwd && want && per_head && p.lds + (size_t)heads * p.split * d * 4 > NR_LDS)
        p.split = 1;
    if (bwd && want)
        p.lds += (size_t)(per_head ? heads * p.split : 8) * d * 4;
    return p;
}

int nr_fill(NrArgs &a, int type, int b, int n, int d, const tpu3_heads *q, const tpu3_heads *k, const void *wq, int wq_head,
            const void *wk, int wk_head, int w_type, const tpu3_positions *pos, float eps, int interleaved)
{
    if (b < 0 || n < 0 || d <= 0 || !hd_type_ok(type) || !hd_type_ok(w_type) || !q || !k || !pos || !(eps >= 0.f))
        return TPU3_EINVAL;
    if (d % 8 || d > 256 || q->heads > 1024 || k->heads > 1024)
        return TPU3_ELIMIT;
    if (q->heads <= 0 || k->heads < 0 || pos->axes < 1 || pos->pairs < 0 || (wq_head != 0 && wq_head != d) ||
        (wk_head != 0 && wk_head != d) || pos->type < TPU3_POS_F32 || pos->type > TPU3_POS_I64 ||
        (pos->freq_type != TPU3_POS_F32 && pos->freq_type != TPU3_POS_F64))
        return TPU3_EINVAL;
    if (pos->axes > d || pos->pairs > d || 2L * pos->axes * pos->pairs > d)
        return TPU3_EINVAL;
    if (b == 0 || n == 0)
        return TPU3_OK;
    if (!hd_rows_ok(q, type) || (k->heads && !hd_rows_ok(k, type)))
        return TPU3_EINVAL;
    if (pos->pairs && (!pos->data || !pos->freq))
        return TPU3_EINVAL;
    if (((uintptr_t)wq & 15) || ((uintptr_t)wk & 15) || (wq && wk && k->heads && (wq_head == 0) != (wk_head == 0)))
        return TPU3_EINVAL;
    a.x[0] = *q, a.x[1] = *k;
    a.w[0] = wq, a.w[1] = k->heads ? wk : nullptr, a.w_head[0] = wq_head, a.w_head[1] = wk_head, a.w_type = w_type;
    a.pos = pos->data, a.pos_type = pos->type, a.pos_sb = pos->sb, a.pos_sn = pos->sr, a.pos_sa = pos->sa;
    a.freq = pos->freq, a.freq_type = pos->freq_type, a.axes = pos->axes, a.pairs = pos->pairs > 0 ? pos->pairs : 1;
    a.total_pairs = pos->axes * pos->pairs;
    a.tokens = (int64_t)b * n, a.n = n, a.d = d, a.interleaved = interleaved != 0;
    a.eps = eps, a.inv_d = 1.f / (float)d;
    return 1;
}

template <typename T> int nr_forward(const NrArgs &a, const NrPlan &p, hipStream_t s)
{
    const dim3 grid((unsigned)((a.tokens + p.tok - 1) / p.tok));
#define NR_GO(L) hipLaunchKernelGGL((norm_rotate_kernel<T, L>), grid, dim3(NR_THREADS), p.lds, s, a)
    if (p.lpr == 4)
        NR_GO(4);
    else if (p.lpr == 8)
        NR_GO(8);
    else if (p.lpr == 16)
        NR_GO(16);
    else
        NR_GO(32);
#undef NR_GO
    return tpu3_launch_status();
}

template <typename T> int nr_backward(const NrArgs &a, const NrPlan &p, hipStream_t s)
{
    const void *f = p.lpr == 4   ? (const void *)norm_rotate_bwd_kernel<T, 4>
                    : p.lpr == 8 ? (const void *)norm_rotate_bwd_kernel<T, 8>
                    : p.lpr == 16 ? (const void *)norm_rotate_bwd_kernel<T, 16>
                                  : (const void *)norm_rotate_bwd_kernel<T, 32>;
    // (the same in every call: another thread's does not lower it)
    const hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)NR_LDS);
    if (e != hipSuccess)
        return (int)e;
#define NR_GO(L) hipLaunchKernelGGL((norm_rotate_bwd_kernel<T, L>), dim3(p.wgs), dim3(NR_THREADS), p.lds, s, a, p.split)
    if (p.lpr == 4)
        NR_GO(4);
    else if (p.lpr == 8)
        NR_GO(8);
    else if (p.lpr == 16)
        NR_GO(16);
    else
        NR_GO(32);
#undef NR_GO
    return tpu3_launch_status();
}

}  // namespace

extern "C" int tpu3_norm_rotate_fwd(tpu3_stream_t stream, int type, int b, int n, int d, const tpu3_heads *q,
                                    const tpu3_heads *k, const void *wq, int wq_head, const void *wk, int wk_head, int w_type,
                                    const tpu3_positions *pos, float eps, int interleaved, void *oq, void *ok)
{
    NrArgs a = {};
    const int rc = nr_fill(a, type, b, n, d, q, k, wq, wq_head, wk, wk_head, w_type, pos, eps, interleaved);
    if (rc <= 0)
        return rc;
    if (!oq || ((uintptr_t)oq & 15) || (k->heads && (!ok || ((uintptr_t)ok & 15))))
        return TPU3_EINVAL;
    a.out[0] = oq, a.out[1] = ok;
    const NrPlan p = nr_plan(a.tokens, q->heads + k->heads, d, a.total_pairs, a.interleaved, false, false, false);
    if ((a.tokens + p.tok - 1) / p.tok >= 1 << 24)              // (2^32 threads a launch)
        return TPU3_ELIMIT;
    a.tok = p.tok;
    const hipStream_t s = (hipStream_t)stream;
    return type == TPU3_TYPE_F32 ? nr_forward<float>(a, p, s) : type == TPU3_TYPE_F16 ? nr_forward<_Float16>(a, p, s) : nr_forward<__bf16>(a, p, s);
}

extern "C" size_t tpu3_norm_rotate_bwd_workspace_bytes(int heads, int d, int per_head)
{
    if (heads <= 0 || d <= 0)
        return 0;
    return (size_t)NR_MAX_WG * (per_head ? heads : 2) * d * 4;
}

extern "C" int tpu3_norm_rotate_bwd(tpu3_stream_t stream, int type, int b, int n, int d, const tpu3_heads *q,
                                    const tpu3_heads *k, const void *wq, int wq_head, const void *wk, int wk_head, int w_type,
                                    const tpu3_positions *pos, float eps, int interleaved, const tpu3_heads *gq,
                                    const tpu3_heads *gk, void *dq, void *dk, void *dwq, void *dwk, void *workspace,
                                    size_t workspace_bytes)
{
    NrArgs a = {};
    const int rc = nr_fill(a, type, b, n, d, q, k, wq, wq_head, wk, wk_head, w_type, pos, eps, interleaved);
    if (rc <= 0)
        return rc;
    if (!hd_rows_ok(gq, type) || gq->heads != q->heads || !dq || ((uintptr_t)dq & 15))
        return TPU3_EINVAL;
    if (k->heads && (!hd_rows_ok(gk, type) || gk->heads != k->heads || !dk || ((uintptr_t)dk & 15)))
        return TPU3_EINVAL;
    a.g[0] = *gq;
    if (k->heads)
        a.g[1] = *gk;
    a.out[0] = dq, a.out[1] = dk;
    a.want_w[0] = dwq && wq, a.want_w[1] = dwk && wk && k->heads;
    const bool want = a.want_w[0] || a.want_w[1], per_head = (wq && wq_head) || (wk && k->heads && wk_head);
    const int heads = q->heads + k->heads;
    if (want && (!workspace || ((uintptr_t)workspace & 3) || workspace_bytes < tpu3_norm_rotate_bwd_workspace_bytes(heads, d, per_head)))
        return TPU3_EINVAL;
    a.part = (float *)workspace;
    const NrPlan p = nr_plan(a.tokens, heads, d, a.total_pairs, a.interleaved, true, per_head, want);
    if (p.lds > NR_LDS)
        return TPU3_ELIMIT;
    a.tok = p.tok;
    const hipStream_t s = (hipStream_t)stream;
    int st = type == TPU3_TYPE_F32 ? nr_backward<float>(a, p, s) : type == TPU3_TYPE_F16 ? nr_backward<_Float16>(a, p, s) : nr_backward<__bf16>(a, p, s);
    if (st || !want)
        return st;
    // columns of a partial row: per head, all query heads' weights then all key heads'; else one set each
    const int cols = (per_head ? heads : 2) * d, nq = (per_head ? q->heads : 1) * d;
    hipLaunchKernelGGL(norm_rotate_wsum_kernel, dim3((cols + NW_COLS - 1) / NW_COLS), dim3(NW_COLS * NW_PARTS), 0, s, p.wgs, cols, nq, w_type,
                       a.part, a.want_w[0] ? dwq : nullptr, a.want_w[1] ? dwk : nullptr);
    return tpu3_launch_status();
}
