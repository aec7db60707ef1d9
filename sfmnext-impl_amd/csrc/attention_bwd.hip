// attention_bwd.hip — gradients of attention.hip (include/sqd.h section 22).
//
//   P = 2^(x - lse),  dP = dO V^T,  dS = P (dP - delta) (1 - tanh^2),  delta_i = dO_i . O_i,
//   gV = P^T dO,  gK = scale dS^T Q,  gQ = scale dS K.
//
// Two kernels and no atomics, so gradients repeat to the bit: one owns 128 keys and walks the rows that see them (gK, gV: four products of
// the row tile), one owns 128 rows and walks their keys (gQ: three products).  Recomputing the scores in both costs 7 products where a single kernel
// with atomic adds into gQ would take 5.
// Measured: 2 x 3840 bf16 in 3 documents, 16 + 4 heads of 128, capped: gK gV 278 us (465 TFLOP/s), gQ 186 us (525); 12 x 480, 12 heads of 64, distance
// bias: 52 and 39 us, row records 10 us; 2 x 1281 fp32, 8 + 4 heads of 40, causal, in 3 parts each: 100 and 76 us.  16 bits: vector pipe 0.38 to 0.55 of
// the time busy (some 15 operations and 1 to 3 exponentials or reciprocals a pair), matrix pipe 0.25 to 0.34, what does not overlap is waited for.
// fp32: matrix pipe 0.56 (gK gV) and 0.67 (gQ).  fp16 on top: the exponents of dS, 5 us, and 2 us of row records.
//
// Roundings of 16-bit types.  dS is packed in two terms, hi and what hi left (2^-16 and finer of it), and gK and gQ take one product more: with one
// term its rounding was as large an error as the gradient's own (1.4 to 2 times the error of one rounding together, 1.0 to 1.2 now).  That product
// and three vector operations a pair cost 12 to 20 % of the two kernels.  P is packed once (gV: 1.4 times one rounding).
//
// P within 2^-22 of one (fp16, whose lse carries the lift's rounding too: 2^-21): every other key's P is below that together and dP - delta is the
// difference of two equal numbers, rounding noise of about that size; dS is taken as zero there.  P of a row that sees ONE key is off by half a unit
// of lse, so such a row has exactly no gradient for its score while |lse| (the score in base 2) is below 8, and noise of (2 D + 64) 2^-24 of
// sum |go v| beyond.  P = 0 (masked): dS is zero whatever dP holds.
#include "attention.h"

namespace sqd {
int attn_check(const char *who, const sqd_attn_args *a);
int attn_check_tensor(const char *who, const char *name, const void *p, const int64_t *stride, int heads, int dtype);
AttnK attn_kargs(const sqd_attn_args *a);
void attn_doc_ranges(const int *ids, int2 *out, int B, int S, int div, int span, int ntile, hipStream_t st);
}  // namespace sqd

namespace {
using namespace sqd;

constexpr int NT = 256, BM = 128;
template <typename T> constexpr float one_less() { return 1.f - (lifted<T>() ? 4.76837158203125e-7f : 2.384185791015625e-7f); }        // 2^-21, 2^-22

// the larger of a value over the 16 groups of 16 lanes (whose lanes agree); `red` 4 floats, valid in every thread
__device__ __forceinline__ float group_max(float v, float *red) {
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    v = fmaxf(v, __shfl_xor(v, 32, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

// What the two gradient kernels read of a packed row, padded to whole tiles: lse, delta = o.go, the last key it may see (-1: none, and then
// its q and go are never loaded), document, and with a bias position and slope.  16 lanes a row, 8 features a lane.  o's rounding alone would be
// as large an error of a gradient as the rounding of dS, so what it left (o_low) is added back.
// fp16: the largest |go|^2 and |delta| of a workgroup's rows, and in workgroups of their own behind those of the rows the largest |v|^2 of 64
// keys, one float each (A.lift_max: [key head][go, delta: a float a row workgroup; v: a float a key workgroup]).
constexpr int VK = 64;
template <typename T>
__global__ __launch_bounds__(NT) void attn_rows_kernel(AttnK A) {
    __shared__ float red[4];
    const int RT = A.Sq * A.G, c = (threadIdx.x & 15) * 8, hk = blockIdx.y, b = blockIdx.z, nr = A.rows_padded / (NT / 16);
    const int64_t bh = (int64_t)b * A.Hkv + hk;
    const int len = A.k_len ? min(max(A.k_len[b], 0), A.Sk) : A.Sk;
    float *lift_max = lifted<T>() ? A.lift_max + bh * (2 * nr + (A.Sk + VK - 1) / VK) : nullptr;
    if (lifted<T>() && (int)blockIdx.x >= nr) {
        const int blk = blockIdx.x - nr;
        float mx = 0.f;
#pragma unroll
        for (int n = 0; n < VK / 16; ++n) {
            const int j = blk * VK + n * 16 + (threadIdx.x >> 4);
            const bool on = j < len && (!A.k_docs || A.k_docs[(int64_t)b * A.Sk + j] >= 0);        // the others hold anything
            float s = 0.f, v[8];
            if (on && c < A.D) {
                load_f32<T, 8>((const T *)A.v + b * A.vs[0] + (int64_t)j * A.vs[1] + hk * A.vs[2] + c, v);
#pragma unroll
                for (int e = 0; e < 8; ++e) s = fmaf(v[e], v[e], s);
            }
#pragma unroll
            for (int k = 8; k > 0; k >>= 1) s += __shfl_xor(s, k, 16);
            mx = fmaxf(mx, s);
        }
        mx = group_max(mx, red);
        if (threadIdx.x == 0) lift_max[2 * nr + blk] = mx;
        return;
    }
    const int R = blockIdx.x * (NT / 16) + (threadIdx.x >> 4);
    const RowOf row = row_of(A, b, R, RT, len, A.prefix ? max(A.prefix[b], 0) : 0);
    const int hq = hk * A.G + row.g;
    const float lse = row.lim >= 0 ? A.lse[bh * RT + R] : INFINITY;
    const bool live = lse != INFINITY;                         // documents may hide every key of a row that its limit allows
    float s = 0.f, g2 = 0.f;
    if (c < A.D && live) {
        const int64_t o = (((int64_t)b * A.Sq + row.i) * A.Hq + hq) * A.D + c;
        float u[8], v[8];
        load_f32<T, 8>((const T *)A.o + o, u);
        if (sizeof(T) == 2 && A.o_low) {
            load_f32<T, 8>((const T *)A.o_low + o, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) u[e] += v[e];
        }
        load_f32<T, 8>((const T *)A.go + b * A.gos[0] + (int64_t)row.i * A.gos[1] + hq * A.gos[2] + c, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(u[e], v[e], s);
        if (lifted<T>())
#pragma unroll
            for (int e = 0; e < 8; ++e) g2 = fmaf(v[e], v[e], g2);
    }
#pragma unroll
    for (int k = 8; k > 0; k >>= 1) {
        s += __shfl_xor(s, k, 16);
        if (lifted<T>()) g2 += __shfl_xor(g2, k, 16);
    }
    if ((threadIdx.x & 15) == 0) {
        const int64_t at = bh * A.rows_padded + R;
        A.row_delta[at] = s;
        A.row_lse[at] = lse;
        A.row_lim[at] = live ? row.lim : -1;
        A.row_doc[at] = row.qd;
        if (A.slopes) {
            A.row_pos[at] = (float)row.pos;
            A.row_slope[at] = A.slopes[hq] * A.unit_inv;
        }
    }
    if (lifted<T>()) {
        const float gm = group_max(g2, red), dm = group_max(fabsf(s), red);
        if (threadIdx.x == 0) lift_max[blockIdx.x] = gm, lift_max[nr + blockIdx.x] = dm;
    }
}

// the exponent of dS, one workgroup a key head; a bound that is no number (or no gradient at all) lifts by nothing
__global__ __launch_bounds__(NT) void attn_lift_kernel(AttnK A) {
    __shared__ float red[3][4];
    const int nr = A.rows_padded / (NT / 16), nv = (A.Sk + VK - 1) / VK, tid = threadIdx.x;
    const float *part = A.lift_max + (int64_t)blockIdx.x * (2 * nr + nv);
    float mx[3] = {0.f, 0.f, 0.f};
    for (int i = tid; i < nr; i += NT) mx[0] = fmaxf(mx[0], part[i]), mx[1] = fmaxf(mx[1], part[nr + i]);
    for (int i = tid; i < nv; i += NT) mx[2] = fmaxf(mx[2], part[2 * nr + i]);
#pragma unroll
    for (int k = 0; k < 3; ++k) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) mx[k] = fmaxf(mx[k], __shfl_xor(mx[k], o, 64));
        if ((tid & 63) == 0) red[k][tid >> 6] = mx[k];
    }
    __syncthreads();
    if (tid) return;
#pragma unroll
    for (int k = 0; k < 3; ++k) mx[k] = fmaxf(fmaxf(red[k][0], red[k][1]), fmaxf(red[k][2], red[k][3]));
    const float bound = sqrtf(mx[0]) * sqrtf(mx[2]) + mx[1];
    A.lift[blockIdx.x] = bound > 0.f && bound < INFINITY ? (float)min(14 - ilogbf(bound), 64) : 0.f;
}

// probability and score gradient (without the scale) of one pair, e = dP - delta; `see` false: zeros, whatever the products hold.  fp16: ds
// comes times `factor` (not by a shift of lse, which would round it)
template <typename T, int CAP, bool BIAS>
__device__ __forceinline__ void pair_grad(float raw, float e, float lse, float slope, float dist, const AttnK &A, bool see, float factor, float &p, float &ds) {
    const float t = CAP ? tanh_of<CAP>(raw, A) : raw, c = CAP ? A.cap_out : A.scale_log2;
    p = exp2_hw(fmaf(BIAS ? fmaf(-slope, fabsf(dist), t) : t, c, -lse));
    p = see ? p : 0.f;
    const float q = see && p < one_less<T>() ? p : 0.f;
    e = see ? (lifted<T>() ? e * factor : e) : 0.f;
    ds = CAP ? q * e * fmaf(-t, t, 1.f) : q * e;
}

// KW waves side by side on 32 keys each, times QW on the 32-row parts of a row tile.  A wave needs its gK and gV sums (64 registers each at 128
// features) and the operands of its keys (32 + 32): with those in registers one wave fits a SIMD and every latency is paid.  KVL keeps the keys'
// operands in LDS instead: at 128 features 8 waves of 256 registers, two a SIMD; at 64 three workgroups of 4 waves a CU.
template <typename T, int DP, int KW, int QW, bool KVL, int CAP, bool BIAS>
__global__ __launch_bounds__(64 * KW * QW, KW * QW == 8 ? 2 : KVL ? 3 : DP * sizeof(T) <= 128 ? 2 : 1) void attn_dkv_kernel(AttnK A) {
    constexpr int NT = 64 * KW * QW, QT = 32 * QW, DB = DP / 32;
    typedef Tile<T, DP> L;
    typedef typename L::frag frag;
    typedef Stage<T, DP, QT, NT> S;
    typedef Stage<T, DP, 32 * KW, NT> SK;
    __shared__ __align__(16) char lrow[4][S::BYTES];           // q, q, go, go
    __shared__ __align__(16) char lk[KVL ? SK::BYTES : 16], lv[KVL ? SK::BYTES : 16];
    __shared__ __align__(16) float rows[2][6 * QT];            // lse, delta, last key, document; with a bias position, slope
    __shared__ int wk[2 * KW];
    static_assert(QW == 1 || sizeof(lrow) >= (size_t)KW * (QW - 1) * 64 * DB * 16 * 4, "a wave's sums fit the row buffers");

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, kw = wave % KW, qw = wave / KW;
    int bh, u0;                                                // the first keys (the most rows, in causal order) first
    if (!dealt(A.deal, blockIdx.x, A.ntile * A.nsplit, bh, u0)) return;
    const int tile = u0 / A.nsplit, split = u0 - tile * A.nsplit, hk = bh % A.Hkv, b = bh / A.Hkv;
    const int RT = A.Sq * A.G, j0 = tile * 32 * KW, jl = j0 + kw * 32 + (lane & 31);
    const int len = A.k_len ? min(max(A.k_len[b], 0), A.Sk) : A.Sk, off = len - A.Sq;
    const int prefix = A.prefix ? max(A.prefix[b], 0) : 0;
    const int *qdoc = A.q_docs ? A.q_docs + (int64_t)b * A.Sq : nullptr;
    const bool docs = qdoc != nullptr;
    int kd = -3;
    if (docs && jl < len) kd = A.k_docs[(int64_t)b * A.Sk + jl];
    const bool on = jl < len && (!docs || kd >= 0);
    if (docs && !on) kd = -3;
    clear_lds<NT>(lrow[0], 4 * S::BYTES, tid);

    int dlo = 0, dhi = 0, wlo = 0, whi = 0;                    // documents of the workgroup's keys, of the wave's
    if (docs) {
        wlo = kd >= 0 ? kd : 0x7fffffff, whi = kd;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            wlo = min(wlo, __shfl_xor(wlo, o, 64));
            whi = max(whi, __shfl_xor(whi, o, 64));
        }
        if (lane == 0 && qw == 0) wk[kw] = wlo, wk[KW + kw] = whi;
    }
    if (KVL) {
        clear_lds<NT>(lk, sizeof(lk), tid);
        clear_lds<NT>(lv, sizeof(lv), tid);
    }
    __syncthreads();
    if (docs) {
        dlo = wk[0], dhi = wk[KW];
#pragma unroll
        for (int k = 1; k < KW; ++k) dlo = min(dlo, wk[k]), dhi = max(dhi, wk[KW + k]);
        dlo = __builtin_amdgcn_readfirstlane(dlo), dhi = __builtin_amdgcn_readfirstlane(dhi);
    }
    int nt = (RT + QT - 1) / QT;
    // rows that see a key >= j0: all of them, in causal order those from query j0 - off on (a prefix past j0: all)
    int t0 = 0;
    if (A.causal && prefix <= j0) t0 = (int)(min((int64_t)max(j0 - off, 0) * A.G, (int64_t)RT) / QT);
    if (j0 >= len) t0 = nt;
    if (A.nsplit > 1) {
        const int per = (nt - t0 + A.nsplit - 1) / A.nsplit;
        t0 = min(nt, t0 + split * per);
        nt = min(nt, t0 + per);
    }
    DocWalk walk(docs ? A.doc_rng + (int64_t)b * A.ndoc_tiles : nullptr, dlo, dhi, nt);
    const bool all_on = __all(on);
    const float jf = (float)jl;
    constexpr float P_UP = lifted<T>() ? P_SCALE : 1.f;
    const float lift = lifted<T>() && RT ? A.lift[bh] : 0.f, factor = ldexpf(1.f, (int)lift);

    frag kf[KVL ? 1 : L::KS], vf[KVL ? 1 : L::KS];
    const T *kbase = (const T *)A.k + b * A.ks[0] + (int64_t)j0 * A.ks[1] + hk * A.ks[2];
    const T *vbase = (const T *)A.v + b * A.vs[0] + (int64_t)j0 * A.vs[1] + hk * A.vs[2];
    if constexpr (KVL) {                                       // padding keys hold anything and are not loaded
        SK sk, sv;
        sk.aim(tid, (unsigned)A.ks[1]);
        sv.aim(tid, (unsigned)A.vs[1]);
        int kp[SK::N];
        if (docs)
#pragma unroll
            for (int n = 0; n < SK::N; ++n) {
                const int r = SK::piece_row(n, tid, A.D);
                kp[n] = r < len - j0 ? A.k_docs[(int64_t)b * A.Sk + j0 + r] : -1;
            }
        sk.load(kbase, lds_offset(lk), tid, A.D, len - j0, docs, kp);
        sv.load(vbase, lds_offset(lv), tid, A.D, len - j0, docs, kp);
    } else {
        const T *krow = kbase + (int64_t)(jl - j0) * A.ks[1], *vrow = vbase + (int64_t)(jl - j0) * A.vs[1];
#pragma unroll
        for (int ks = 0; ks < L::KS; ++ks) {
            kf[ks] = L::mem_frag(krow, ks, h, A.D, on);
            vf[ks] = L::mem_frag(vrow, ks, h, A.D, on);
        }
    }

    const T *qb = (const T *)A.q + b * A.qs[0] + (int64_t)hk * A.G * A.qs[2], *gb = (const T *)A.go + b * A.gos[0] + (int64_t)hk * A.G * A.gos[2];
    const int64_t row_at = (int64_t)bh * A.rows_padded;
    S sq, sg;
    sq.aim_packed(tid, 0, A.G, A.g_magic, (unsigned)A.qs[1], (unsigned)A.qs[2]);
    sg.aim_packed(tid, 0, A.G, A.g_magic, (unsigned)A.gos[1], (unsigned)A.gos[2]);
    const unsigned oq = lds_offset(lrow[0]), og = oq + 2 * S::BYTES, orow = lds_offset(rows[0]);
    // rows that see no key hold anything and are not loaded: their limits are read a tile ahead of the DMA that goes by them
    const bool skips = docs || (A.causal && off < 0 && prefix <= 0);
    int pd[S::N];
    auto peek = [&](int t) {
        if (!skips) return;
#pragma unroll
        for (int n = 0; n < S::N; ++n) {
            const int r = S::piece_row(n, tid, A.D);
            pd[n] = t < nt && r < RT - t * QT ? A.row_lim[row_at + t * QT + r] : -1;
        }
    };
    auto fetch = [&](int t, int s) {
        const int i0 = div_g(t * QT, A.g_magic), rem = t * QT - i0 * A.G;
        if (QT % A.G) {                                        // otherwise a tile starts with head 0 and the offsets are those of the first tile
            sq.aim_packed(tid, rem, A.G, A.g_magic, (unsigned)A.qs[1], (unsigned)A.qs[2]);
            sg.aim_packed(tid, rem, A.G, A.g_magic, (unsigned)A.gos[1], (unsigned)A.gos[2]);
        }
        sq.load(qb + i0 * A.qs[1], oq + s * S::BYTES, tid, A.D, RT - t * QT, skips, pd);
        sg.load(gb + i0 * A.gos[1], og + s * S::BYTES, tid, A.D, RT - t * QT, skips, pd);
        if (wave == 3) {                                       // QT / 4 lanes an array
            const int k = lane / (QT / 4), e = lane % (QT / 4) * 16;
            const int64_t d1 = (const char *)A.row_delta - (const char *)A.row_lse;              // the arrays follow each other, d1 bytes apart
            if (k < 4) dma16(A.row_lse + row_at + t * QT, (unsigned)(k * d1) + e, orow + s * 24 * QT);
            if (BIAS && k < 2) dma16(A.row_pos + row_at + t * QT, (unsigned)(k * d1) + e, orow + s * 24 * QT + 16 * QT);
        }
    };

    f32x16 gk[DB], gv[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) gk[db] = f32x16{}, gv[db] = f32x16{};
    int s = 0;
    bool u, un;
    int t = walk.next(t0, u);
    peek(t);
    if (t < nt) fetch(t, 0);
    int tn = walk.next(t + 1, un);
    peek(tn);
    dma_wait();
    __syncthreads();
    // Two waves of a SIMD that meet at one barrier a tile do their products at the same time and their exponentials at the same time.  With
    // 8 waves the second four run half a tile behind: two barriers a tile, the first four pass [products, half of the pairs] while the others pass
    // [half of the pairs, products].  A tile's buffer is then free half a tile later, so the first four fetch in mid-tile; the loads of either
    // have the half tile up to the same barrier.
    constexpr bool STAGGER = KW * QW == 8;
    const bool late = STAGGER && qw == 1;
    auto meet = [] {                                           // (this wave's reads of the buffers that the meeting frees have come back)
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0xc07f);                    // lgkmcnt(0)
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    if (late) meet();
    while (t < nt) {
        if ((!STAGGER || late) && tn < nt) fetch(tn, s ^ 1);
        const int q0 = qw * 32;
        const float *rw = rows[s];
        const char *lq = lrow[s], *lg = lrow[2 + s];
        f32x16 xs[1] = {f32x16{}}, dps[1];                     // dP starts from -delta
        f32x16 &x = xs[0], &dp = dps[0];
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            const f32x4 d = *reinterpret_cast<const f32x4 *>(rw + QT + q0 + 8 * r4 + 4 * h);
#pragma unroll
            for (int e = 0; e < 4; ++e) dp[4 * r4 + e] = -d[e];
        }
        constexpr int BATCH = KVL ? 2 : batch_of<T, L::KS>();
        product<T, 1, L::KS, BATCH>(xs, A.D, [&](int, int ks) { return L::row_frag(lq, q0 + (lane & 31), ks, h); },
                                    [&](int ks) { return KVL ? L::row_frag(lk, kw * 32 + (lane & 31), ks, h) : kf[KVL ? 0 : ks]; });
        product<T, 1, L::KS, BATCH>(dps, A.D, [&](int, int ks) { return L::row_frag(lg, q0 + (lane & 31), ks, h); },
                                    [&](int ks) { return KVL ? L::row_frag(lv, kw * 32 + (lane & 31), ks, h) : vf[KVL ? 0 : ks]; });
        // every row of the tile sees all of the wave's keys?  (limits do not fall with the row)
        const int R0 = t * QT + q0;
        const bool part = !all_on || !u || R0 + 32 > RT || row_limit(div_g(R0, A.g_magic) + off, len, A.causal, prefix) < j0 + kw * 32 + 31;
        // 8 registers (16 rows of the tile) at a time: probabilities and score gradients, then their shares of gV and gK.  The second half's pairs
        // run under the first half's products.
        float p[8], ds[8];
        auto pairs = [&](auto half, auto masked) {
#pragma unroll
            for (int r2 = 0; r2 < 2; ++r2) {
                constexpr int H = decltype(half)::value;
                const int q4 = q0 + 8 * (2 * H + r2) + 4 * h;
                const f32x4 lse = *reinterpret_cast<const f32x4 *>(rw + q4);
                int4 lim = make_int4(0, 0, 0, 0), qd = make_int4(kd, kd, kd, kd);
                f32x4 ps = {0, 0, 0, 0}, sl = {0, 0, 0, 0};
                if (masked) lim = *reinterpret_cast<const int4 *>(rw + 2 * QT + q4);
                if (masked && docs) qd = *reinterpret_cast<const int4 *>(rw + 3 * QT + q4);
                if (BIAS) ps = *reinterpret_cast<const f32x4 *>(rw + 4 * QT + q4), sl = *reinterpret_cast<const f32x4 *>(rw + 5 * QT + q4);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = (2 * H + r2) * 4 + e;
                    const int le = e == 0 ? lim.x : e == 1 ? lim.y : e == 2 ? lim.z : lim.w, de = e == 0 ? qd.x : e == 1 ? qd.y : e == 2 ? qd.z : qd.w;
                    pair_grad<T, CAP, BIAS>(x[r], dp[r], lse[e], sl[e], ps[e] - jf, A, !masked || (jl <= le && de == kd), factor, p[r2 * 4 + e],
                                                      ds[r2 * 4 + e]);
                    if (lifted<T>()) p[r2 * 4 + e] *= P_UP;
                }
            }
        };
        auto grads = [&](auto half) {
            if (part) pairs(half, std::true_type{});
            else pairs(half, std::false_type{});
        };
        frag cg[DB], cq[DB], pf, df, dl;
        auto operands = [&](int row) {
#pragma unroll
            for (int db = 0; db < DB; ++db) cg[db] = L::col_frag(lg, q0 + row, db, lane);
#pragma unroll
            for (int db = 0; db < DB; ++db) cq[db] = L::col_frag(lq, q0 + row, db, lane);
        };
        auto products = [&] {
#pragma unroll
            for (int db = 0; db < DB; ++db) gv[db] = Mma<T>::mma(cg[db], pf, gv[db]);
#pragma unroll
            for (int db = 0; db < DB; ++db) gk[db] = Mma<T>::mma(cq[db], df, gk[db]);
            if constexpr (sizeof(T) == 2)
#pragma unroll
                for (int db = 0; db < DB; ++db) gk[db] = Mma<T>::mma(cq[db], dl, gk[db]);
        };
        auto packed = [&] {
            pf = Mma<T>::pack(p), df = Mma<T>::pack(ds);
            if constexpr (sizeof(T) == 2) dl = Mma<T>::rest(ds, df);
        };
        grads(std::integral_constant<int, 0>{});
        packed();
        if (STAGGER) {
            if (late) dma_wait();
            meet();
            if (!late && tn < nt) fetch(tn, s ^ 1);
        }
        bool u2 = true;
        const int t2 = walk.next(tn + 1, u2);
        peek(t2);
        operands(0);
        __builtin_amdgcn_sched_barrier(0);
        products();
        grads(std::integral_constant<int, 1>{});
        packed();
        operands(16);
        __builtin_amdgcn_sched_barrier(0);
        products();
        if (STAGGER) {
            if (!late) dma_wait();
            meet();
        } else {
            dma_wait();
            __syncthreads();
        }
        s ^= 1;
        t = tn, u = un, tn = t2, un = u2;
    }
    if (STAGGER && !late) meet();
    __syncthreads();
    if (QW > 1) {                                              // the row halves' sums, through the row buffers: gK, then gV
        float *red = reinterpret_cast<float *>(lrow[0]);
        auto join = [&](f32x16 (&g)[DB]) {
            if (qw > 0)
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int r = 0; r < 16; ++r) red[(((qw - 1) * KW + kw) * DB * 16 + db * 16 + r) * 64 + lane] = g[db][r];
            __syncthreads();
            if (qw == 0)
#pragma unroll
                for (int k = 0; k < QW - 1; ++k)
#pragma unroll
                    for (int db = 0; db < DB; ++db)
#pragma unroll
                        for (int r = 0; r < 16; ++r) g[db][r] += red[((k * KW + kw) * DB * 16 + db * 16 + r) * 64 + lane];
            __syncthreads();
        };
        join(gk);
        join(gv);
        if (qw > 0) return;
    }
    if (jl >= A.Sk) return;
    const int64_t o = (((int64_t)b * A.Sk + jl) * A.Hkv + hk) * A.D;
    const float ku = lifted<T>() ? ldexpf(A.scale, -(int)lift) : A.scale, vu = 1.f / P_UP;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            const int d = db * 32 + 8 * r4 + 4 * h;
            if (d >= A.D) continue;
            const float a[4] = {gk[db][4 * r4] * ku, gk[db][4 * r4 + 1] * ku, gk[db][4 * r4 + 2] * ku, gk[db][4 * r4 + 3] * ku};
            const float c[4] = {gv[db][4 * r4] * vu, gv[db][4 * r4 + 1] * vu, gv[db][4 * r4 + 2] * vu, gv[db][4 * r4 + 3] * vu};
            if (A.nsplit > 1) {
                const int64_t at = (int64_t)split * A.B * A.Sk * A.Hkv * A.D + o + d;
                store_f32<float, 4>(A.part_a + at, a);
                store_f32<float, 4>(A.part_b + at, c);
                continue;
            }
            store_f32<T, 4>((T *)A.gk + o + d, a);
            store_f32<T, 4>((T *)A.gv + o + d, c);
        }
}

template <typename T, int DP, int CAP, bool BIAS>
__global__ __launch_bounds__(NT, sizeof(T) == 4 && DP == 128 ? 1 : 2) void attn_dq_kernel(AttnK A) {
    constexpr int KT = 32, DB = DP / 32;
    typedef Tile<T, DP> L;
    typedef typename L::frag frag;
    typedef Stage<T, DP, KT, NT> S;
    __shared__ __align__(16) char lk[2][S::BYTES], lv[2][S::BYTES];
    __shared__ __align__(16) int ld[2][KT];
    __shared__ int wq[8];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    int bh, w;
    if (!dealt(A.deal, blockIdx.x, A.ntile * A.nsplit, bh, w)) return;
    const int split = w % A.nsplit, tile = A.ntile - 1 - w / A.nsplit, hk = bh % A.Hkv, b = bh / A.Hkv;
    const int RT = A.Sq * A.G, row0 = tile * BM;
    const int len = A.k_len ? min(max(A.k_len[b], 0), A.Sk) : A.Sk;
    const int prefix = A.prefix ? max(A.prefix[b], 0) : 0;
    const int R = row0 + wave * 32 + (lane & 31);
    const RowOf row = row_of(A, b, R, RT, len, prefix);
    clear_lds<NT>(lk[0], 2 * S::BYTES, tid);
    clear_lds<NT>(lv[0], 2 * S::BYTES, tid);
    int kend = len;
    if (A.causal) kend = max(0, min(len, max(min(A.Sq - 1, div_g(row0 + BM - 1, A.g_magic)) + len - A.Sq + 1, prefix)));
    int dlo = 0, dhi = 0;
    if (A.q_docs) {
        int lo = row.qd >= 0 ? row.qd : 0x7fffffff, hi = row.qd;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            lo = min(lo, __shfl_xor(lo, o, 64));
            hi = max(hi, __shfl_xor(hi, o, 64));
        }
        if (lane == 0) wq[wave] = lo, wq[4 + wave] = hi;
    }
    __syncthreads();
    if (A.q_docs) {
        dlo = __builtin_amdgcn_readfirstlane(min(min(wq[0], wq[1]), min(wq[2], wq[3])));
        dhi = __builtin_amdgcn_readfirstlane(max(max(wq[4], wq[5]), max(wq[6], wq[7])));
    }
    const int nt_all = (kend + KT - 1) / KT, per = (nt_all + A.nsplit - 1) / A.nsplit, t0 = min(nt_all, split * per), t1 = min(nt_all, t0 + per);
    DocWalk walk(A.q_docs ? A.doc_rng + (int64_t)b * A.ndoc_tiles : nullptr, dlo, dhi, t1);

    frag qf[L::KS], gf[L::KS];
    const int64_t rec = (int64_t)bh * A.rows_padded + R;
    const bool live = row.on && A.row_lim[rec] >= 0;           // rows that see no key (documents may hide every key of a row's limit) hold anything
    const T *qrow = (const T *)A.q + b * A.qs[0] + (int64_t)row.i * A.qs[1] + (int64_t)(hk * A.G + row.g) * A.qs[2];
    const T *grow = (const T *)A.go + b * A.gos[0] + (int64_t)row.i * A.gos[1] + (int64_t)(hk * A.G + row.g) * A.gos[2];
#pragma unroll
    for (int ks = 0; ks < L::KS; ++ks) {
        qf[ks] = L::mem_frag(qrow, ks, h, A.D, live);
        gf[ks] = L::mem_frag(grow, ks, h, A.D, live);
    }
    float lse = INFINITY, delta = 0.f;
    if (live) lse = A.row_lse[rec], delta = A.row_delta[rec];
    const float lift = lifted<T>() ? A.lift[bh] : 0.f, factor = ldexpf(1.f, (int)lift);

    const T *kbase = (const T *)A.k + b * A.ks[0] + hk * A.ks[2], *vbase = (const T *)A.v + b * A.vs[0] + hk * A.vs[2];
    const int *kdoc = A.k_docs ? A.k_docs + (int64_t)b * A.Sk : nullptr;
    S sk, sv;
    sk.aim(tid, (unsigned)A.ks[1]);
    sv.aim(tid, (unsigned)A.vs[1]);
    const unsigned ok = lds_offset(lk[0]), ov = lds_offset(lv[0]);
    int pd[S::N], sd = -1;                                     // as in the forward
    auto peek = [&](int t) {
        if (!kdoc) return;
#pragma unroll
        for (int n = 0; n < S::N; ++n) {
            const int r = S::piece_row(n, tid, A.D);
            pd[n] = t < t1 && r < len - t * KT ? kdoc[t * KT + r] : -1;
        }
        sd = t < t1 && tid < KT && t * KT + tid < len ? kdoc[t * KT + tid] : -1;
    };
    auto fetch = [&](int t, int s) {
        const int64_t j0 = (int64_t)t * KT;
        sk.load(kbase + j0 * A.ks[1], ok + s * S::BYTES, tid, A.D, len - t * KT, kdoc != nullptr, pd);
        sv.load(vbase + j0 * A.vs[1], ov + s * S::BYTES, tid, A.D, len - t * KT, kdoc != nullptr, pd);
        if (kdoc && tid < KT) ld[s][tid] = sd;
    };
    const float slope = BIAS && row.on ? A.slopes[hk * A.G + row.g] * A.unit_inv : 0.f;
    f32x16 gq[DB], minus_delta;                                // dP starts from -delta: 16 registers against 16 subtractions a step
#pragma unroll
    for (int db = 0; db < DB; ++db) gq[db] = f32x16{};
#pragma unroll
    for (int r = 0; r < 16; ++r) minus_delta[r] = -delta;

    int s = 0;
    bool u, un;
    int t = walk.next(t0, u);
    peek(t);
    if (t < t1) fetch(t, 0);
    int tn = walk.next(t + 1, un);
    peek(tn);
    dma_wait();
    __syncthreads();
    while (t < t1) {
        if (tn < t1) fetch(tn, s ^ 1);
        bool u2 = true;
        const int t2 = walk.next(tn + 1, u2);
        peek(t2);
        const int j0 = t * KT;
        f32x16 xs[1] = {f32x16{}}, dps[1] = {minus_delta};
        f32x16 &x = xs[0], &dp = dps[0];
        product<T, 1, L::KS, batch_of<T, L::KS>()>(xs, A.D, [&](int, int ks) { return L::row_frag(lk[s], lane & 31, ks, h); }, [&](int ks) { return qf[ks]; });
        product<T, 1, L::KS, batch_of<T, L::KS>()>(dps, A.D, [&](int, int ks) { return L::row_frag(lv[s], lane & 31, ks, h); }, [&](int ks) { return gf[ks]; });
        const bool part = !u || __any(row.lim < j0 + KT - 1);
        float ds[16];
        const float d0 = (float)(row.pos - j0 - 4 * h);
        auto grads = [&](auto masked) {
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                const int j4 = 8 * r4 + 4 * h;
                int4 kd = make_int4(row.qd, row.qd, row.qd, row.qd);
                if (masked && kdoc) kd = *reinterpret_cast<const int4 *>(&ld[s][j4]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = r4 * 4 + e, j = j0 + j4 + e, d = e == 0 ? kd.x : e == 1 ? kd.y : e == 2 ? kd.z : kd.w;
                    float p;
                    pair_grad<T, CAP, BIAS>(x[r], dp[r], lse, slope, d0 - (float)(8 * r4 + e), A, !masked || (j <= row.lim && d == row.qd), factor, p, ds[r]);
                }
            }
        };
        if (part) grads(std::true_type{});
        else grads(std::false_type{});
        frag cf[2][DB];
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
            for (int db = 0; db < DB; ++db) cf[kk][db] = L::col_frag(lk[s], kk * 16, db, lane);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            const frag df = Mma<T>::pack(&ds[8 * kk]);
#pragma unroll
            for (int db = 0; db < DB; ++db) gq[db] = Mma<T>::mma(cf[kk][db], df, gq[db]);
            if constexpr (sizeof(T) == 2) {
                const frag dl = Mma<T>::rest(&ds[8 * kk], df);
#pragma unroll
                for (int db = 0; db < DB; ++db) gq[db] = Mma<T>::mma(cf[kk][db], dl, gq[db]);
            }
        }
        dma_wait();
        __syncthreads();
        s ^= 1;
        t = tn, u = un, tn = t2, un = u2;
    }
    if (!row.on) return;
    const int64_t out = (((int64_t)b * A.Sq + row.i) * A.Hq + hk * A.G + row.g) * A.D;
    const float qu = lifted<T>() ? ldexpf(A.scale, -(int)lift) : A.scale;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            const int d = db * 32 + 8 * r4 + 4 * h;
            const float v[4] = {gq[db][4 * r4] * qu, gq[db][4 * r4 + 1] * qu, gq[db][4 * r4 + 2] * qu, gq[db][4 * r4 + 3] * qu};
            if (d >= A.D) continue;
            if (A.nsplit > 1) store_f32<float, 4>(A.part_a + (int64_t)split * A.B * A.Sq * A.Hq * A.D + out + d, v);
            else store_f32<T, 4>((T *)A.gq + out + d, v);
        }
}

// out = the parts of a gradient, added in order
template <typename T>
__global__ __launch_bounds__(NT) void attn_parts_kernel(const float *__restrict__ part, T *__restrict__ out, int64_t n4, int nsplit) {
    const int64_t u = (int64_t)blockIdx.x * NT + threadIdx.x;
    if (u >= n4) return;
    float a[4];
    load_f32<float, 4>(part + u * 4, a);
    for (int s = 1; s < nsplit; ++s) {
        float b[4];
        load_f32<float, 4>(part + (s * n4 + u) * 4, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] += b[e];
    }
    store_f32<T, 4>(out + u * 4, a);
}

struct BwdPlan { int kw, qw, rows_padded, nq_tiles, nk_tiles, k_split, q_split, nv; int64_t rows, nk, nq, lift, parts, scratch; };
// parts of the looped-over side (of the whole side, documents or not): with fewer than 192 workgroups CUs idle, and 512 shorter ones also even out
// causal rows (168 of fp32, 1281 tokens: dK dV 214 -> 108 us in 3 parts); at least 8 tiles each.  With 240 (3 documents, 3840 tokens) parts lose: 306 -> 493 us, documents being uneven in them.
int parts_of(int64_t blocks, int64_t tiles) {
    int64_t n = blocks && blocks < 192 ? 512 / blocks : 1;
    n = n > tiles / 8 ? tiles / 8 : n;
    return (int)(n < 1 ? 1 : n > 16 ? 16 : n);
}
BwdPlan bwd_plan(const sqd_attn_args *a) {
    BwdPlan p{};
    const int G = a->Hq / a->Hkv;
    // keys and row parts of a workgroup.  128 x 2 with 8 waves where that fits (16-bit types past 64 features) and most CUs get one.  Else 4 waves: 64
    // x 2 makes twice the workgroups of 128 x 1, which wins once those fill the card by themselves (measured with dS in one term, at two sizes a
    // type: bf16, 64 features: 576 workgroups of 128 keys 47 us against 56, 480: 58 against 54; fp32: 768: 482 against 500, 576: 259 against 242)
    const int64_t wide = (int64_t)((a->Sk + 127) / 128) * a->B * a->Hkv;
    if (a->dtype != SQD_F32 && a->D > 64 && wide >= 192) p.kw = 4, p.qw = 2;
    else if (wide < (a->dtype == SQD_F32 ? 768 : 512)) p.kw = 2, p.qw = 2;
    else p.kw = 4, p.qw = 1;
    const int QT = 32 * p.qw;
    p.rows_padded = (a->Sq * G + 63) / 64 * 64;
    p.rows = (int64_t)a->B * a->Hkv * p.rows_padded;
    p.nq_tiles = a->q_docs ? (a->Sq * G + QT - 1) / QT : 0;
    p.nk_tiles = a->q_docs ? (a->Sk + 31) / 32 : 0;
    p.nk = (int64_t)a->B * a->Sk * a->Hkv * a->D, p.nq = (int64_t)a->B * a->Sq * a->Hq * a->D;
    p.k_split = parts_of((int64_t)((a->Sk + 32 * p.kw - 1) / (32 * p.kw)) * a->B * a->Hkv, (a->Sq * G + QT - 1) / QT);
    p.q_split = parts_of((int64_t)((a->Sq * G + BM - 1) / BM) * a->B * a->Hkv, (a->Sk + 31) / 32);
    const int64_t pk = p.k_split > 1 ? 2 * p.k_split * p.nk : 0, pq = p.q_split > 1 ? p.q_split * p.nq : 0;      // one after the other
    p.nv = a->dtype == SQD_F16 ? (a->Sk + VK - 1) / VK : 0;                        // (fp16: the exponents and the maxima they come from)
    p.lift = (a->slopes ? 6 : 4) * p.rows + ((int64_t)2 * a->B * (p.nq_tiles + p.nk_tiles) + 3) / 4 * 4;
    p.parts = p.lift + (a->dtype == SQD_F16 ? ((int64_t)a->B * a->Hkv * (1 + 2 * (p.rows_padded / (NT / 16)) + p.nv) + 3) / 4 * 4 : 0);
    p.scratch = p.parts + (pk > pq ? pk : pq);
    return p;
}
}  // namespace

extern "C" int64_t sqd_attn_bwd_scratch(const sqd_attn_args *a) {
    if (sqd::attn_check("sqd_attn_bwd_scratch", a)) return SQD_EINVAL;
    return bwd_plan(a).scratch;
}

extern "C" int sqd_attn_bwd(const sqd_attn_args *a) {
    using namespace sqd;
    const char *who = "sqd_attn_bwd";
    if (int e = attn_check(who, a)) return e;
    if (a->B == 0 || (a->Sq == 0 && a->Sk == 0)) return SQD_OK;
    if (a->Sq) {
        if (int e = attn_check_tensor(who, "q", a->q, a->q_stride, a->Hq, a->dtype)) return e;
        if (int e = attn_check_tensor(who, "go", a->go, a->go_stride, a->Hq, a->dtype)) return e;
        SQD_CHECK_ARG(a->o && aligned16(a->o) && aligned16(a->o_low) && aligned16(a->gq) && a->lse && a->scratch && aligned16(a->scratch),
                      "%s: null or unaligned pointer", who);
    }
    if (a->Sk) {
        if (int e = attn_check_tensor(who, "k", a->k, a->k_stride, a->Hkv, a->dtype)) return e;
        if (int e = attn_check_tensor(who, "v", a->v, a->v_stride, a->Hkv, a->dtype)) return e;
        SQD_CHECK_ARG(!a->gk == !a->gv && aligned16(a->gk) && aligned16(a->gv), "%s: gk and gv come together, 16-byte aligned", who);
    }
    const BwdPlan p = bwd_plan(a);
    SQD_CHECK_ARG(p.rows < (1 << 28) && a->B < 65536 && a->Hkv < 65536, "%s: too many tokens", who);          // row records: 32-bit offsets between arrays
    const int nk_wg = (a->Sk + 32 * p.kw - 1) / (32 * p.kw), nq_wg = (int)(((int64_t)a->Sq * (a->Hq / a->Hkv) + BM - 1) / BM);
    SQD_CHECK_ARG(p.rows_padded / (NT / 16) + p.nv <= max_blocks(NT) && (int64_t)a->B * a->Hkv * (nk_wg + 8) * p.k_split < (1 << 30) &&
                      (int64_t)a->B * a->Hkv * (nq_wg + 8) * p.q_split < (1 << 30) &&
                      deal_blocks(deal(a->B * a->Hkv, nk_wg * p.k_split)) <= max_blocks(64 * p.kw * p.qw) &&
                      deal_blocks(deal(a->B * a->Hkv, nq_wg * p.q_split)) <= max_blocks(NT), "%s: too many tokens", who);
    AttnK A = attn_kargs(a);
    A.rows_padded = p.rows_padded;
    A.row_lse = a->scratch, A.row_delta = a->scratch + p.rows;
    A.row_lim = (int *)(a->scratch + 2 * p.rows), A.row_doc = (int *)(a->scratch + 3 * p.rows);
    A.row_pos = a->scratch + 4 * p.rows, A.row_slope = a->scratch + 5 * p.rows;
    int2 *q_rng = reinterpret_cast<int2 *>(a->scratch + (a->slopes ? 6 : 4) * p.rows), *k_rng = q_rng + (int64_t)a->B * p.nq_tiles;
    A.lift = a->scratch + p.lift, A.lift_max = A.lift + (int64_t)a->B * a->Hkv;
    const hipStream_t st = (hipStream_t)a->stream;
    return for_dtype(a->dtype, [&](auto tt) {
        using T = decltype(tt);
        if (p.rows) hipLaunchKernelGGL((attn_rows_kernel<T>), dim3(p.rows_padded / (NT / 16) + p.nv, A.Hkv, A.B), dim3(NT), 0, st, A);
        if (p.rows && lifted<T>()) hipLaunchKernelGGL(attn_lift_kernel, dim3(A.B * A.Hkv), dim3(NT), 0, st, A);
        if (p.nq_tiles) attn_doc_ranges(A.q_docs, q_rng, A.B, A.Sq, A.G, 32 * p.qw, p.nq_tiles, st);
        if (p.nk_tiles) attn_doc_ranges(A.k_docs, k_rng, A.B, A.Sk, 1, 32, p.nk_tiles, st);
        auto go = [&](auto dp, auto cap, auto bias) {
            constexpr int DP = decltype(dp)::value;
            constexpr int CAP = decltype(cap)::value;
            constexpr bool BIAS = decltype(bias)::value;
            if (A.Sk && A.gk) {
                AttnK K = A;
                K.ntile = nk_wg, K.doc_rng = q_rng, K.ndoc_tiles = p.nq_tiles;
                K.nsplit = p.k_split, K.part_a = a->scratch + p.parts, K.part_b = K.part_a + p.k_split * p.nk;
                K.deal = deal(A.B * A.Hkv, K.ntile * K.nsplit);
                const dim3 grid((unsigned)deal_blocks(K.deal));
                if (p.kw == 2) hipLaunchKernelGGL((attn_dkv_kernel<T, DP, 2, 2, false, CAP, BIAS>), grid, dim3(NT), 0, st, K);
                else if constexpr (sizeof(T) == 2 && DP == 128) hipLaunchKernelGGL((attn_dkv_kernel<T, DP, 4, 2, true, CAP, BIAS>), grid, dim3(512), 0, st, K);
                else hipLaunchKernelGGL((attn_dkv_kernel<T, DP, 4, 1, (DP * sizeof(T) == 128), CAP, BIAS>), grid, dim3(NT), 0, st, K);
                if (K.nsplit > 1) {                                // (parts of dK, dV are joined before the scratch holds dQ's)
                    const dim3 g2((unsigned)((p.nk / 4 + NT - 1) / NT));
                    hipLaunchKernelGGL((attn_parts_kernel<T>), g2, dim3(NT), 0, st, K.part_a, (T *)a->gk, p.nk / 4, K.nsplit);
                    hipLaunchKernelGGL((attn_parts_kernel<T>), g2, dim3(NT), 0, st, K.part_b, (T *)a->gv, p.nk / 4, K.nsplit);
                }
            }
            if (A.Sq && A.gq) {
                AttnK Q = A;
                Q.ntile = nq_wg, Q.doc_rng = k_rng, Q.ndoc_tiles = p.nk_tiles;
                Q.nsplit = p.q_split, Q.part_a = a->scratch + p.parts;
                Q.deal = deal(A.B * A.Hkv, Q.ntile * Q.nsplit);
                hipLaunchKernelGGL((attn_dq_kernel<T, DP, CAP, BIAS>), dim3((unsigned)deal_blocks(Q.deal)), dim3(NT), 0, st, Q);
                if (Q.nsplit > 1)
                    hipLaunchKernelGGL((attn_parts_kernel<T>), dim3((unsigned)((p.nq / 4 + NT - 1) / NT)), dim3(NT), 0, st, Q.part_a, (T *)a->gq, p.nq / 4, Q.nsplit);
            }
        };
        auto flags = [&](auto dp) { for_scores<T>(cap_form(a->softcap, a->dtype), a->slopes != nullptr, [&](auto cap, auto bias) { go(dp, cap, bias); }); };
        if (a->D <= 32) flags(std::integral_constant<int, 32>{});
        else if (a->D <= 64) flags(std::integral_constant<int, 64>{});
        else flags(std::integral_constant<int, 128>{});
        SQD_CHECK_LAUNCH("sqd_attn_bwd");
        return SQD_OK;
    });
}
