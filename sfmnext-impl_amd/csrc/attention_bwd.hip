// attention_bwd.hip — gradients of attention.hip (include/sqd.h section 22).
//
//   P = 2^(x - lse),  dP = dO V^T,  dS = P (dP - delta) (1 - tanh^2),  delta_i = dO_i . O_i,
//   gV = P^T dO,  gK = scale dS^T Q,  gQ = scale dS K.
//
// Two kernels and no atomics, so gradients repeat to the bit: one owns 128 keys and walks the rows that see them (gK, gV: four products of
// the row tile), one owns 128 rows and walks their keys (gQ: three products).  Recomputing the scores in both costs 7 products where a single kernel
// with atomic adds into gQ would take 5.
//
// P within 2^-22 of one: every other key's P is below 2^-22 together and dP - delta is the difference of two equal numbers, rounding noise of
// about that size; dS is taken as zero there (a row that sees ONE key has exactly no gradient for its scores).  P = 0 (masked): dS is zero
// whatever dP holds.
#include "attention.h"

namespace sqd {
int attn_check(const char *who, const sqd_attn_args *a);
int attn_check_tensor(const char *who, const char *name, const void *p, const int64_t *stride, int dtype);
AttnK attn_kargs(const sqd_attn_args *a);
void attn_doc_ranges(const int *ids, int2 *out, int B, int S, int div, int span, int ntile, hipStream_t st);
}  // namespace sqd

namespace {
using namespace sqd;

constexpr int NT = 256, BM = 128;
constexpr float ONE_LESS = 1.f - 2.384185791015625e-7f;        // 1 - 2^-22

// delta [B,Hkv,Sq*G] (packed rows): 16 lanes a row, 8 features a lane
template <typename T>
__global__ __launch_bounds__(NT) void attn_delta_kernel(AttnK A) {
    const int RT = A.Sq * A.G, c = (threadIdx.x & 15) * 8;
    const int64_t at = (int64_t)blockIdx.x * (NT / 16) + (threadIdx.x >> 4), rows = (int64_t)A.B * A.Hkv * RT;
    if (at >= rows) return;
    const int64_t bh = at / RT;
    const int R = (int)(at - bh * RT), i = R / A.G, hq = (int)(bh % A.Hkv) * A.G + R - i * A.G;
    const int64_t b = bh / A.Hkv;
    float s = 0.f;
    if (c < A.D) {
        float u[8], v[8];
        load_f32<T, 8>((const T *)A.o + ((b * A.Sq + i) * A.Hq + hq) * A.D + c, u);
        load_f32<T, 8>((const T *)A.go + b * A.gos[0] + i * A.gos[1] + hq * A.gos[2] + c, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(u[e], v[e], s);
    }
#pragma unroll
    for (int k = 8; k > 0; k >>= 1) s += __shfl_xor(s, k, 16);
    if ((threadIdx.x & 15) == 0) A.delta[at] = s;
}

// one score's probability and the factor 1 - tanh^2
template <bool CAP, bool BIAS> __device__ __forceinline__ float score(float raw, const AttnK &A, float slope, float dist, float &fac) {
    float x;
    fac = 1.f;
    if (CAP) {
        const float t = tanh_of<CAP>(raw, A.cap_in);
        fac = fmaf(-t, t, 1.f);
        x = A.cap_out * t;
    } else {
        x = raw;                                               // the scale goes into the exponent's fma
    }
    if (BIAS) x = fmaf(-slope, fabsf(dist), CAP ? x : x * A.scale_log2);
    return x;
}

template <typename T, int DP, bool CAP, bool BIAS>
__global__ __launch_bounds__(NT, 1) void attn_dkv_kernel(AttnK A) {
    constexpr int QT = 32, DB = DP / 32;
    typedef Tile<T, DP> L;
    typedef typename L::frag frag;
    __shared__ __align__(16) char lq[2][QT * L::PITCH], lg[2][QT * L::PITCH];
    __shared__ __align__(16) float r_lse[2][QT], r_delta[2][QT], r_slope[2][QT];
    __shared__ __align__(16) int r_lim[2][QT], r_doc[2][QT], r_pos[2][QT];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    int w = xcd_order(blockIdx.x, gridDim.x);
    const int tile = w % A.ntile, bh = w / A.ntile, hk = bh % A.Hkv, b = bh / A.Hkv;
    const int RT = A.Sq * A.G, j0 = tile * 128, jl = j0 + wave * 32 + (lane & 31);
    const int len = A.k_len ? min(max(A.k_len[b], 0), A.Sk) : A.Sk, off = len - A.Sq;
    const int prefix = A.prefix ? A.prefix[b] : 0;
    const bool docs = A.k_docs != nullptr;
    int kd = -1;
    if (docs && jl < len) kd = A.k_docs[(int64_t)b * A.Sk + jl];
    const bool on = jl < len && (!docs || kd >= 0);
    if (docs && !on) kd = -3;

    int dlo = 0, dhi = 0;
    if (docs) {                                                // documents of the 128 keys: the four ranges of 32
        __shared__ int wk[8];
        int lo = kd >= 0 ? kd : 0x7fffffff, hi = kd;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            lo = min(lo, __shfl_xor(lo, o, 64));
            hi = max(hi, __shfl_xor(hi, o, 64));
        }
        if (lane == 0) wk[wave] = lo, wk[4 + wave] = hi;
        __syncthreads();
        dlo = min(min(wk[0], wk[1]), min(wk[2], wk[3]));
        dhi = max(max(wk[4], wk[5]), max(wk[6], wk[7]));
    }
    const int2 *rng = A.doc_rng + (int64_t)b * A.ndoc_tiles;
    const int nt = (RT + QT - 1) / QT;
    // rows that see a key >= j0: all of them, in causal order those from query j0 - off on (a prefix past j0: all)
    int t0 = 0;
    if (A.causal && prefix <= j0) t0 = (int)(min((int64_t)max(j0 - off, 0) * A.G, (int64_t)RT) / QT);
    if (j0 >= len) t0 = nt;
    auto next = [&](int t) {
        if (docs)
            while (t < nt && (rng[t].y < dlo || rng[t].x > dhi)) ++t;
        return t;
    };

    frag kf[L::KS], vf[L::KS];
    const T *krow = (const T *)A.k + b * A.ks[0] + (int64_t)jl * A.ks[1] + hk * A.ks[2];
    const T *vrow = (const T *)A.v + b * A.vs[0] + (int64_t)jl * A.vs[1] + hk * A.vs[2];
#pragma unroll
    for (int ks = 0; ks < L::KS; ++ks) {
        kf[ks] = L::mem_frag(krow, ks, h, A.D, on);
        vf[ks] = L::mem_frag(vrow, ks, h, A.D, on);
    }

    const T *qb = (const T *)A.q + b * A.qs[0] + (int64_t)hk * A.G * A.qs[2], *gb = (const T *)A.go + b * A.gos[0] + (int64_t)hk * A.G * A.gos[2];
    Stage<T, DP, QT, NT> sq, sg;
    float s_lse = 0.f, s_delta = 0.f, s_slope = 0.f;
    int s_lim = -1, s_doc = -2, s_pos = 0;
    auto fetch = [&](int t) {
        auto row_of = [&](const T *base, const int64_t *st) {
            const int64_t s1 = st[1], s2 = st[2];
            return [=, &A](int r) -> const T * {
                const int R = t * QT + r;
                if (R >= RT) return nullptr;
                const int i = R / A.G, g = R - i * A.G;
                if (docs && A.q_docs[(int64_t)b * A.Sq + i] < 0) return nullptr;        // rows that see no key hold anything
                if (row_limit(i + off, len, A.causal, prefix) < 0) return nullptr;
                return base + i * s1 + g * s2;
            };
        };
        sq.load(tid, A.D, row_of(qb, A.qs));
        sg.load(tid, A.D, row_of(gb, A.gos));
        if (tid < QT) {
            const int R = t * QT + tid;
            s_lim = -1, s_doc = -2, s_lse = INFINITY, s_delta = 0.f;
            if (R < RT) {
                const int i = R / A.G;
                s_pos = i + off;
                s_lse = A.lse[(int64_t)bh * RT + R];
                s_delta = A.delta[(int64_t)bh * RT + R];
                if (BIAS) s_slope = A.slopes[hk * A.G + R - i * A.G] * 1.44269504088896341f;
                if (docs) s_doc = A.q_docs[(int64_t)b * A.Sq + i];
                if (!docs || s_doc >= 0) s_lim = row_limit(s_pos, len, A.causal, prefix);
            }
        }
    };
    auto put = [&](int s) {
        sq.store(lq[s], tid);
        sg.store(lg[s], tid);
        if (tid < QT) {
            r_lse[s][tid] = s_lse, r_delta[s][tid] = s_delta, r_lim[s][tid] = s_lim, r_doc[s][tid] = s_doc, r_pos[s][tid] = s_pos;
            if (BIAS) r_slope[s][tid] = s_slope;
        }
    };

    f32x16 gk[DB], gv[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) gk[db] = f32x16{}, gv[db] = f32x16{};
    int t = next(t0), s = 0;
    if (t < nt) {
        fetch(t);
        put(0);
    }
    __syncthreads();
    while (t < nt) {
        const int tn = next(t + 1);
        if (tn < nt) fetch(tn);
        f32x16 x = {}, dp = {};
#pragma unroll
        for (int ks = 0; ks < L::KS; ++ks) {
            x = Mma<T>::mma(L::row_frag(lq[s], lane & 31, ks, h), kf[ks], x);
            dp = Mma<T>::mma(L::row_frag(lg[s], lane & 31, ks, h), vf[ks], dp);
        }
        float p[16], ds[16];
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            const int q4 = 8 * r4 + 4 * h;
            const f32x4 lse = *reinterpret_cast<const f32x4 *>(&r_lse[s][q4]), delta = *reinterpret_cast<const f32x4 *>(&r_delta[s][q4]);
            const int4 lim = *reinterpret_cast<const int4 *>(&r_lim[s][q4]);
            int4 qd = make_int4(kd, kd, kd, kd), ps = make_int4(0, 0, 0, 0);
            f32x4 sl = {0, 0, 0, 0};
            if (docs) qd = *reinterpret_cast<const int4 *>(&r_doc[s][q4]);
            if (BIAS) ps = *reinterpret_cast<const int4 *>(&r_pos[s][q4]), sl = *reinterpret_cast<const f32x4 *>(&r_slope[s][q4]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = r4 * 4 + e;
                const int le = e == 0 ? lim.x : e == 1 ? lim.y : e == 2 ? lim.z : lim.w, de = e == 0 ? qd.x : e == 1 ? qd.y : e == 2 ? qd.z : qd.w;
                const int pe = e == 0 ? ps.x : e == 1 ? ps.y : e == 2 ? ps.z : ps.w;
                float fac;
                const float v = score<CAP, BIAS>(x[r], A, sl[e], (float)(pe - jl), fac);
                const bool see = jl <= le && de == kd;
                p[r] = see ? exp2_hw(fmaf(v, CAP || BIAS ? 1.f : A.scale_log2, -lse[e])) : 0.f;
                ds[r] = p[r] > 0.f && p[r] < ONE_LESS ? p[r] * (dp[r] - delta[e]) * fac : 0.f;
            }
        }
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            const frag pf = Mma<T>::pack(&p[8 * kk]), df = Mma<T>::pack(&ds[8 * kk]);
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                gv[db] = Mma<T>::mma(L::col_frag(lg[s], kk * 16, db, lane), pf, gv[db]);
                gk[db] = Mma<T>::mma(L::col_frag(lq[s], kk * 16, db, lane), df, gk[db]);
            }
        }
        if (tn < nt) put(s ^ 1);
        __syncthreads();
        s ^= 1;
        t = tn;
    }
    if (jl >= A.Sk) return;
    const int64_t o = (((int64_t)b * A.Sk + jl) * A.Hkv + hk) * A.D;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            const int d = db * 32 + 8 * r4 + 4 * h;
            if (d >= A.D) continue;
            const float a[4] = {gk[db][4 * r4] * A.scale, gk[db][4 * r4 + 1] * A.scale, gk[db][4 * r4 + 2] * A.scale, gk[db][4 * r4 + 3] * A.scale};
            const float c[4] = {gv[db][4 * r4], gv[db][4 * r4 + 1], gv[db][4 * r4 + 2], gv[db][4 * r4 + 3]};
            store_f32<T, 4>((T *)A.gk + o + d, a);
            store_f32<T, 4>((T *)A.gv + o + d, c);
        }
}

template <typename T, int DP, bool CAP, bool BIAS>
__global__ __launch_bounds__(NT, sizeof(T) == 4 && DP == 128 ? 1 : 2) void attn_dq_kernel(AttnK A) {
    constexpr int KT = 32, DB = DP / 32;
    typedef Tile<T, DP> L;
    typedef typename L::frag frag;
    __shared__ __align__(16) char lk[2][KT * L::PITCH], lv[2][KT * L::PITCH];
    __shared__ __align__(16) int ld[2][KT];
    __shared__ int wq[8];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    int w = xcd_order(blockIdx.x, gridDim.x);
    const int tile = A.ntile - 1 - w % A.ntile, bh = w / A.ntile, hk = bh % A.Hkv, b = bh / A.Hkv;
    const int RT = A.Sq * A.G, row0 = tile * BM;
    const int len = A.k_len ? min(max(A.k_len[b], 0), A.Sk) : A.Sk, off = len - A.Sq;
    const int prefix = A.prefix ? A.prefix[b] : 0;
    const int R = row0 + wave * 32 + (lane & 31);
    const bool in = R < RT;
    const int i = in ? R / A.G : A.Sq - 1, g = in ? R - i * A.G : 0, pos = i + off;
    int qd = -2;
    if (A.q_docs && in) qd = max(A.q_docs[(int64_t)b * A.Sq + i], -2);
    if (qd < 0) qd = -2;
    const bool on = in && (!A.q_docs || qd >= 0);
    const int lim = on ? row_limit(pos, len, A.causal, prefix) : -1;
    int kend = len;
    if (A.causal) kend = max(0, min(len, max(min(A.Sq - 1, (row0 + BM - 1) / A.G) + off + 1, prefix)));
    int dlo = 0, dhi = 0;
    if (A.q_docs) {
        int lo = qd >= 0 ? qd : 0x7fffffff, hi = qd;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            lo = min(lo, __shfl_xor(lo, o, 64));
            hi = max(hi, __shfl_xor(hi, o, 64));
        }
        if (lane == 0) wq[wave] = lo, wq[4 + wave] = hi;
        __syncthreads();
        dlo = min(min(wq[0], wq[1]), min(wq[2], wq[3]));
        dhi = max(max(wq[4], wq[5]), max(wq[6], wq[7]));
    }
    const int t1 = (kend + KT - 1) / KT;
    // the ranges are those of 64 keys
    const int2 *rng = A.doc_rng + (int64_t)b * A.ndoc_tiles;
    auto next = [&](int t) {
        if (A.q_docs)
            while (t < t1 && (rng[t].y < dlo || rng[t].x > dhi)) ++t;
        return t;
    };

    frag qf[L::KS], gf[L::KS];
    const T *qrow = (const T *)A.q + b * A.qs[0] + (int64_t)i * A.qs[1] + (int64_t)(hk * A.G + g) * A.qs[2];
    const T *grow = (const T *)A.go + b * A.gos[0] + (int64_t)i * A.gos[1] + (int64_t)(hk * A.G + g) * A.gos[2];
#pragma unroll
    for (int ks = 0; ks < L::KS; ++ks) {
        qf[ks] = L::mem_frag(qrow, ks, h, A.D, on);
        gf[ks] = L::mem_frag(grow, ks, h, A.D, on);
    }
    float lse = INFINITY, delta = 0.f;
    if (on) lse = A.lse[(int64_t)bh * RT + R], delta = A.delta[(int64_t)bh * RT + R];

    const T *kbase = (const T *)A.k + b * A.ks[0] + hk * A.ks[2], *vbase = (const T *)A.v + b * A.vs[0] + hk * A.vs[2];
    const int *kdoc = A.k_docs ? A.k_docs + (int64_t)b * A.Sk : nullptr;
    Stage<T, DP, KT, NT> sk, sv;
    int sd = -1;
    auto fetch = [&](int t) {
        const int j0 = t * KT;
        auto row_of = [&](const T *base, int64_t stride) {
            return [=](int r) -> const T * {
                const int j = j0 + r;
                if (j >= len || (kdoc && kdoc[j] < 0)) return nullptr;
                return base + j * stride;
            };
        };
        sk.load(tid, A.D, row_of(kbase, A.ks[1]));
        sv.load(tid, A.D, row_of(vbase, A.vs[1]));
        if (kdoc && tid < KT) sd = j0 + tid < len ? kdoc[j0 + tid] : -1;
    };
    auto put = [&](int s) {
        sk.store(lk[s], tid);
        sv.store(lv[s], tid);
        if (kdoc && tid < KT) ld[s][tid] = sd;
    };
    const float slope = BIAS && in ? A.slopes[hk * A.G + g] * 1.44269504088896341f : 0.f;
    f32x16 gq[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) gq[db] = f32x16{};

    int t = next(0), s = 0;
    if (t < t1) {
        fetch(t);
        put(0);
    }
    __syncthreads();
    while (t < t1) {
        const int tn = next(t + 1);
        if (tn < t1) fetch(tn);
        const int j0 = t * KT;
        f32x16 x = {}, dp = {};
#pragma unroll
        for (int ks = 0; ks < L::KS; ++ks) {
            x = Mma<T>::mma(L::row_frag(lk[s], lane & 31, ks, h), qf[ks], x);
            dp = Mma<T>::mma(L::row_frag(lv[s], lane & 31, ks, h), gf[ks], dp);
        }
        float ds[16];
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            const int j4 = 8 * r4 + 4 * h;
            int4 kd = make_int4(qd, qd, qd, qd);
            if (kdoc) kd = *reinterpret_cast<const int4 *>(&ld[s][j4]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = r4 * 4 + e, j = j0 + j4 + e, d = e == 0 ? kd.x : e == 1 ? kd.y : e == 2 ? kd.z : kd.w;
                float fac;
                const float v = score<CAP, BIAS>(x[r], A, slope, (float)(pos - j), fac);
                const float p = j <= lim && d == qd ? exp2_hw(fmaf(v, CAP || BIAS ? 1.f : A.scale_log2, -lse)) : 0.f;
                ds[r] = p > 0.f && p < ONE_LESS ? p * (dp[r] - delta) * fac : 0.f;
            }
        }
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            const frag df = Mma<T>::pack(&ds[8 * kk]);
#pragma unroll
            for (int db = 0; db < DB; ++db) gq[db] = Mma<T>::mma(L::col_frag(lk[s], kk * 16, db, lane), df, gq[db]);
        }
        if (tn < t1) put(s ^ 1);
        __syncthreads();
        s ^= 1;
        t = tn;
    }
    if (!in) return;
    T *out = (T *)A.gq + (((int64_t)b * A.Sq + i) * A.Hq + hk * A.G + g) * A.D;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            const int d = db * 32 + 8 * r4 + 4 * h;
            const float v[4] = {gq[db][4 * r4] * A.scale, gq[db][4 * r4 + 1] * A.scale, gq[db][4 * r4 + 2] * A.scale, gq[db][4 * r4 + 3] * A.scale};
            if (d < A.D) store_f32<T, 4>(out + d, v);
        }
}

struct BwdPlan { int64_t rows; int nq_tiles, nk_tiles; int64_t delta, q_rng, k_rng; };
BwdPlan bwd_plan(const sqd_attn_args *a) {
    BwdPlan p{};
    const int G = a->Hq / a->Hkv;
    p.rows = (int64_t)a->B * a->Hkv * a->Sq * G;
    p.nq_tiles = a->q_docs ? (a->Sq * G + 31) / 32 : 0;
    p.nk_tiles = a->q_docs ? (a->Sk + 31) / 32 : 0;
    p.delta = (p.rows + 3) / 4 * 4;
    p.q_rng = (int64_t)2 * a->B * p.nq_tiles;
    p.k_rng = (int64_t)2 * a->B * p.nk_tiles;
    return p;
}
}  // namespace

extern "C" int64_t sqd_attn_bwd_scratch(const sqd_attn_args *a) {
    if (sqd::attn_check("sqd_attn_bwd_scratch", a)) return SQD_EINVAL;
    const BwdPlan p = bwd_plan(a);
    return p.delta + p.q_rng + p.k_rng;
}

extern "C" int sqd_attn_bwd(const sqd_attn_args *a) {
    using namespace sqd;
    const char *who = "sqd_attn_bwd";
    if (int e = attn_check(who, a)) return e;
    if (a->B == 0 || (a->Sq == 0 && a->Sk == 0)) return SQD_OK;
    if (a->Sq) {
        if (int e = attn_check_tensor(who, "q", a->q, a->q_stride, a->dtype)) return e;
        if (int e = attn_check_tensor(who, "go", a->go, a->go_stride, a->dtype)) return e;
        SQD_CHECK_ARG(a->o && aligned16(a->o) && a->gq && aligned16(a->gq) && a->lse && a->scratch && aligned16(a->scratch), "%s: null or unaligned pointer", who);
    }
    if (a->Sk) {
        if (int e = attn_check_tensor(who, "k", a->k, a->k_stride, a->dtype)) return e;
        if (int e = attn_check_tensor(who, "v", a->v, a->v_stride, a->dtype)) return e;
        SQD_CHECK_ARG(a->gk && a->gv && aligned16(a->gk) && aligned16(a->gv), "%s: null or unaligned pointer", who);
    }
    const BwdPlan p = bwd_plan(a);
    AttnK A = attn_kargs(a);
    A.delta = a->scratch;
    int2 *q_rng = reinterpret_cast<int2 *>(a->scratch + p.delta), *k_rng = q_rng + (int64_t)a->B * p.nq_tiles;
    const hipStream_t st = (hipStream_t)a->stream;
    return for_dtype(a->dtype, [&](auto tt) {
        using T = decltype(tt);
        if (p.rows) hipLaunchKernelGGL((attn_delta_kernel<T>), dim3((unsigned)((p.rows + 15) / 16)), dim3(NT), 0, st, A);
        if (p.nq_tiles) attn_doc_ranges(A.q_docs, q_rng, A.B, A.Sq, A.G, 32, p.nq_tiles, st);
        if (p.nk_tiles) attn_doc_ranges(A.k_docs, k_rng, A.B, A.Sk, 1, 32, p.nk_tiles, st);
        auto go = [&](auto dp, auto cap, auto bias) {
            constexpr int DP = decltype(dp)::value;
            constexpr bool CAP = decltype(cap)::value, BIAS = decltype(bias)::value;
            if (A.Sk) {
                AttnK K = A;
                K.ntile = (A.Sk + 127) / 128, K.doc_rng = q_rng, K.ndoc_tiles = p.nq_tiles;
                hipLaunchKernelGGL((attn_dkv_kernel<T, DP, CAP, BIAS>), dim3((unsigned)((int64_t)K.ntile * A.B * A.Hkv)), dim3(NT), 0, st, K);
            }
            if (A.Sq) {
                AttnK Q = A;
                Q.ntile = (int)(((int64_t)A.Sq * A.G + BM - 1) / BM), Q.doc_rng = k_rng, Q.ndoc_tiles = p.nk_tiles;
                hipLaunchKernelGGL((attn_dq_kernel<T, DP, CAP, BIAS>), dim3((unsigned)((int64_t)Q.ntile * A.B * A.Hkv)), dim3(NT), 0, st, Q);
            }
        };
        auto flags = [&](auto dp) {
            const bool cap = a->softcap > 0.f, bias = a->slopes != nullptr;
            if (cap && bias) go(dp, std::true_type{}, std::true_type{});
            else if (cap) go(dp, std::true_type{}, std::false_type{});
            else if (bias) go(dp, std::false_type{}, std::true_type{});
            else go(dp, std::false_type{}, std::false_type{});
        };
        if (a->D <= 32) flags(std::integral_constant<int, 32>{});
        else if (a->D <= 64) flags(std::integral_constant<int, 64>{});
        else flags(std::integral_constant<int, 128>{});
        SQD_CHECK_LAUNCH("sqd_attn_bwd");
        return SQD_OK;
    });
}
