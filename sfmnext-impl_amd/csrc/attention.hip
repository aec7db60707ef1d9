// attention.hip — attention forward for packed / causal / prefix / cached tokens with capped scores and a bias by distance (include/sqd.h
// section 22).  o = softmax(z) v over the keys a row may see, one pass over the keys with a running maximum and sum (fp32, base 2).
#include "attention.h"

namespace {
using namespace sqd;

constexpr int NT = 256, BM = 128;       // four waves of 32 rows

// smallest and largest document id of each tile of `span` entries (a negative id anywhere: smallest = -1, so the tile is never taken for a
// uniform one); `div` entries of the tile index share one id (packed query rows: G)
__global__ __launch_bounds__(64) void doc_range_kernel(const int *__restrict__ ids, int2 *__restrict__ out, int S, int div, int span, int ntile) {
    const int b = blockIdx.y, t = blockIdx.x;
    int lo = 0x7fffffff, hi = -1;
    const int e0 = t * span / div, e1 = min(S - 1, ((t + 1) * span - 1) / div);
    for (int e = e0 + (int)threadIdx.x; e <= e1; e += 64) {
        const int d = max(ids[(int64_t)b * S + e], -1);
        lo = min(lo, d);
        hi = max(hi, d);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        lo = min(lo, __shfl_xor(lo, o, 64));
        hi = max(hi, __shfl_xor(hi, o, 64));
    }
    if (threadIdx.x == 0) out[(int64_t)b * ntile + t] = make_int2(lo, hi);
}

template <typename T, int DP, int KT, bool CAP, bool BIAS>
__global__ __launch_bounds__(NT, sizeof(T) == 4 && DP == 128 ? 1 : 2) void attn_fwd_kernel(AttnK A) {
    typedef Tile<T, DP> L;
    typedef typename L::frag frag;
    constexpr int NB = KT / 32, DB = DP / 32;
    __shared__ __align__(16) char lk[2][KT * L::PITCH], lv[2][KT * L::PITCH];
    __shared__ __align__(16) int ld[2][KT];
    __shared__ int wq[8];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    int w = xcd_order(blockIdx.x, gridDim.x);
    const int tile = A.ntile - 1 - w % A.ntile;                 // the longest causal rows first
    w /= A.ntile;
    const int split = w % A.nsplit, bh = w / A.nsplit, hk = bh % A.Hkv, b = bh / A.Hkv;
    const int RT = A.Sq * A.G, row0 = tile * BM;
    const int len = A.k_len ? min(max(A.k_len[b], 0), A.Sk) : A.Sk, off = len - A.Sq;
    const int prefix = A.prefix ? A.prefix[b] : 0;

    // this lane's row (both half-waves hold the same 32 rows)
    const int R = row0 + wave * 32 + (lane & 31);
    const bool on = R < RT;
    const int i = on ? R / A.G : A.Sq - 1, g = on ? R - i * A.G : 0, pos = i + off;
    int qd = -2;
    if (A.q_docs && on) {
        qd = A.q_docs[(int64_t)b * A.Sq + i];
        if (qd < 0) qd = -2;
    }
    const int lim = on && qd != -2 || (on && !A.q_docs) ? row_limit(pos, len, A.causal, prefix) : -1;

    // keys any row of the workgroup may see
    int kend = len;
    if (A.causal) kend = max(0, min(len, max(min(A.Sq - 1, (row0 + BM - 1) / A.G) + off + 1, prefix)));
    int dlo = 0x7fffffff, dhi = -1;
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
    const int nt_all = (kend + KT - 1) / KT, per = (nt_all + A.nsplit - 1) / A.nsplit;
    const int t0 = min(nt_all, split * per), t1 = min(nt_all, t0 + per);
    const int2 *rng = A.doc_rng + (int64_t)b * A.ndoc_tiles;
    auto next = [&](int t) {
        if (A.q_docs)
            while (t < t1 && (rng[t].y < dlo || rng[t].x > dhi)) ++t;
        return t;
    };

    frag qf[L::KS];
    const T *qrow = (const T *)A.q + b * A.qs[0] + (int64_t)i * A.qs[1] + (int64_t)(hk * A.G + g) * A.qs[2];
#pragma unroll
    for (int ks = 0; ks < L::KS; ++ks) qf[ks] = L::mem_frag(qrow, ks, h, A.D, on);

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

    const float slope = BIAS && on ? A.slopes[hk * A.G + g] * 1.44269504088896341f : 0.f;
    f32x16 o[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db] = f32x16{};
    float m = -INFINITY, l = 0.f;

    int t = next(t0), s = 0;
    if (t < t1) {
        fetch(t);
        put(0);
    }
    __syncthreads();
    while (t < t1) {
        const int tn = next(t + 1);
        if (tn < t1) fetch(tn);
        const int j0 = t * KT;

        f32x16 x[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            x[nb] = f32x16{};
#pragma unroll
            for (int ks = 0; ks < L::KS; ++ks) x[nb] = Mma<T>::mma(L::row_frag(lk[s], nb * 32 + (lane & 31), ks, h), qf[ks], x[nb]);
        }
        if (CAP || BIAS) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    float v = CAP ? A.cap_out * tanh_of<CAP>(x[nb][r], A.cap_in) : x[nb][r] * A.scale_log2;
                    if (BIAS) v = fmaf(-slope, fabsf((float)(pos - (j0 + nb * 32 + (r & 3) + 8 * (r >> 2) + 4 * h))), v);
                    x[nb][r] = v;
                }
        }
        const float c = CAP || BIAS ? 1.f : A.scale_log2;
        // the mask, where a row of the wave does not see the whole tile
        bool part = __any(lim < j0 + KT - 1);
        if (kdoc) part = part || !(dlo == dhi && rng[t].x == dlo && rng[t].y == dlo);
        if (part) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) {
                    const int j4 = nb * 32 + 8 * r4 + 4 * h;
                    int4 kd = make_int4(qd, qd, qd, qd);
                    if (kdoc) kd = *reinterpret_cast<const int4 *>(&ld[s][j4]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int d = e == 0 ? kd.x : e == 1 ? kd.y : e == 2 ? kd.z : kd.w;
                        if (j0 + j4 + e > lim || d != qd) x[nb][r4 * 4 + e] = -INFINITY;
                    }
                }
        }
        float mx = x[0][0];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = fmaxf(mx, x[nb][r]);
        const float mn = fmaxf(m, half_max(mx) * c), base = mn == -INFINITY ? 0.f : mn;
        if (__any(mn > m)) {
            const float alpha = exp2_hw(m - base);
            l *= alpha;
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
            m = mn;
        }
        float p[NB][16];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                p[nb][r] = exp2_hw(fmaf(x[nb][r], c, -base));
                l += p[nb][r];
            }
        // P is rounded to the values' type for the second product (half a step of that type, relative); the sum keeps the unrounded P
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                const frag pf = Mma<T>::pack(&p[nb][8 * kk]);
#pragma unroll
                for (int db = 0; db < DB; ++db) o[db] = Mma<T>::mma(L::col_frag(lv[s], nb * 32 + kk * 16, db, lane), pf, o[db]);
            }
        if (tn < t1) put(s ^ 1);
        __syncthreads();
        s ^= 1;
        t = tn;
    }

    l = half_sum(l);
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    if (!on) return;
    const int64_t at = (int64_t)bh * RT + R;
    if (A.nsplit > 1) {
        float *po = A.part_o + ((int64_t)split * A.B * A.Hkv * RT + at) * A.D;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                const int d = db * 32 + 8 * r4 + 4 * h;
                const float v[4] = {o[db][4 * r4] * inv, o[db][4 * r4 + 1] * inv, o[db][4 * r4 + 2] * inv, o[db][4 * r4 + 3] * inv};
                if (d < A.D) store_f32<float, 4>(po + d, v);
            }
        if (h == 0) A.part_lse[(int64_t)split * A.B * A.Hkv * RT + at] = l == 0.f ? -INFINITY : m + __builtin_amdgcn_logf(l);
        return;
    }
    T *out = (T *)A.o + (((int64_t)b * A.Sq + i) * A.Hq + hk * A.G + g) * A.D;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            const int d = db * 32 + 8 * r4 + 4 * h;
            const float v[4] = {o[db][4 * r4] * inv, o[db][4 * r4 + 1] * inv, o[db][4 * r4 + 2] * inv, o[db][4 * r4 + 3] * inv};
            if (d < A.D) store_f32<T, 4>(out + d, v);
        }
    if (A.lse && h == 0) A.lse[at] = l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l);
}

// joins the parts of a row: weights 2^(lse_s - max), added in order of the parts.  One thread per 4 features.
template <typename T>
__global__ __launch_bounds__(NT) void attn_join_kernel(AttnK A) {
    const int RT = A.Sq * A.G, D4 = A.D / 4;
    const int64_t rows = (int64_t)A.B * A.Hkv * RT, u = (int64_t)blockIdx.x * NT + threadIdx.x;
    if (u >= rows * D4) return;
    const int64_t at = u / D4;
    const int d = (int)(u - at * D4) * 4;
    float mx = -INFINITY;
    for (int s = 0; s < A.nsplit; ++s) mx = fmaxf(mx, A.part_lse[s * rows + at]);
    const float base = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f, a[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < A.nsplit; ++s) {
        const float lse = A.part_lse[s * rows + at];
        if (lse == -INFINITY) continue;
        const float wgt = exp2_hw(lse - base);
        sum += wgt;
        float v[4];
        load_f32<float, 4>(A.part_o + (s * rows + at) * A.D + d, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = fmaf(wgt, v[e], a[e]);
    }
    const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] *= inv;
    const int64_t bh = at / RT;
    const int R = (int)(at - bh * RT), i = R / A.G, g = R - i * A.G, hk = (int)(bh % A.Hkv);
    store_f32<T, 4>((T *)A.o + (((bh / A.Hkv) * A.Sq + i) * A.Hq + hk * A.G + g) * A.D + d, a);
    if (A.lse && d == 0) A.lse[at] = sum == 0.f ? INFINITY : mx + __builtin_amdgcn_logf(sum);
}

template <typename T> constexpr int key_tile() { return sizeof(T) == 4 ? 32 : 64; }
int pad_dim(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }

struct Split { int nsplit, ndoc_tiles; int64_t part_floats, lse_floats, rng_floats; };
Split plan(const sqd_attn_args *a) {
    const int KT = a->dtype == SQD_F32 ? 32 : 64, G = a->Hq / a->Hkv;
    const int64_t rows = (int64_t)a->Sq * G, groups = (int64_t)a->B * a->Hkv * ((rows + BM - 1) / BM);
    Split p{};
    // two workgroups fit a CU: split the keys while fewer than 512 would run, down to 4 key tiles (256 keys) for each
    const int tiles = (a->Sk + KT - 1) / KT;
    int64_t n = groups ? 512 / groups : 1;
    n = n > tiles / 4 ? tiles / 4 : n;
    p.nsplit = (int)(n < 1 ? 1 : n > 64 ? 64 : n);
    p.ndoc_tiles = a->q_docs ? tiles : 0;
    p.part_floats = p.nsplit > 1 ? (int64_t)p.nsplit * a->B * a->Hkv * rows * a->D : 0;
    p.lse_floats = p.nsplit > 1 ? ((int64_t)p.nsplit * a->B * a->Hkv * rows + 3) / 4 * 4 : 0;
    p.rng_floats = (int64_t)2 * a->B * p.ndoc_tiles;
    return p;
}
}  // namespace

namespace sqd {
int attn_check(const char *who, const sqd_attn_args *a) {
    SQD_CHECK_ARG(a, "%s: null argument block", who);
    SQD_CHECK_ARG(a->B >= 0 && a->Sq >= 0 && a->Sk >= 0 && a->Hq > 0 && a->Hkv > 0 && a->Hq % a->Hkv == 0, "%s: bad shape B=%d Sq=%d Sk=%d Hq=%d Hkv=%d",
                  who, a->B, a->Sq, a->Sk, a->Hq, a->Hkv);
    SQD_CHECK_ARG(a->D >= 8 && a->D <= 128 && a->D % 8 == 0, "%s: %d features a head (a multiple of 8 up to 128)", who, a->D);
    SQD_CHECK_ARG(a->Sk < (1 << 24) && (int64_t)a->Sq * (a->Hq / a->Hkv) < (1 << 30) && (int64_t)a->B * a->Hkv < (1 << 24), "%s: too many tokens", who);
    SQD_CHECK_ARG(a->scale > 0.f && a->scale < 3e38f && a->softcap >= 0.f && a->softcap < 3e38f, "%s: scale %g, cap %g", who, (double)a->scale, (double)a->softcap);
    SQD_CHECK_ARG(a->dtype >= SQD_F32 && a->dtype <= SQD_F16, "%s: element type %d", who, a->dtype);
    SQD_CHECK_ARG(!a->prefix || a->causal, "%s: a prefix needs the causal order", who);
    SQD_CHECK_ARG(!a->q_docs == !a->k_docs, "%s: documents of queries and keys come together", who);
    return SQD_OK;
}
int attn_check_tensor(const char *who, const char *name, const void *p, const int64_t *stride, int dtype) {
    const int V = dtype == SQD_F32 ? 4 : 8;
    SQD_CHECK_ARG(p && aligned16(p) && stride[0] % V == 0 && stride[1] % V == 0 && stride[2] % V == 0, "%s: %s must be 16-byte aligned, its strides too", who, name);
    return SQD_OK;
}
AttnK attn_kargs(const sqd_attn_args *a) {
    AttnK A{};
    A.q = a->q, A.k = a->k, A.v = a->v, A.go = a->go, A.o = a->o, A.gq = a->gq, A.gk = a->gk, A.gv = a->gv, A.lse = a->lse;
    A.slopes = a->slopes, A.prefix = a->prefix, A.q_docs = a->q_docs, A.k_docs = a->k_docs, A.k_len = a->k_len;
    for (int i = 0; i < 3; ++i) A.qs[i] = a->q_stride[i], A.ks[i] = a->k_stride[i], A.vs[i] = a->v_stride[i], A.gos[i] = a->go_stride[i];
    constexpr double LOG2E = 1.44269504088896340736;
    A.scale = a->scale;
    A.scale_log2 = (float)(a->scale * LOG2E);
    if (a->softcap > 0.f) A.cap_in = (float)(2.0 * LOG2E * a->scale / a->softcap), A.cap_out = (float)(a->softcap * LOG2E);
    A.B = a->B, A.Sq = a->Sq, A.Sk = a->Sk, A.Hq = a->Hq, A.Hkv = a->Hkv, A.G = a->Hq / a->Hkv, A.D = a->D, A.causal = a->causal;
    return A;
}
void attn_doc_ranges(const int *ids, int2 *out, int B, int S, int div, int span, int ntile, hipStream_t st) {
    hipLaunchKernelGGL(doc_range_kernel, dim3(ntile, B), dim3(64), 0, st, ids, out, S, div, span, ntile);
}
}  // namespace sqd

extern "C" int64_t sqd_attn_fwd_scratch(const sqd_attn_args *a) {
    if (attn_check("sqd_attn_fwd_scratch", a)) return SQD_EINVAL;
    if ((int64_t)a->B * a->Sq == 0) return 0;
    const Split p = plan(a);
    return p.part_floats + p.lse_floats + p.rng_floats;
}

extern "C" int sqd_attn_fwd(const sqd_attn_args *a) {
    if (int e = attn_check("sqd_attn_fwd", a)) return e;
    if ((int64_t)a->B * a->Sq == 0) return SQD_OK;
    SQD_CHECK_ARG(a->o && aligned16(a->o), "sqd_attn_fwd: o must be 16-byte aligned");
    if (int e = attn_check_tensor("sqd_attn_fwd", "q", a->q, a->q_stride, a->dtype)) return e;
    if (a->Sk) {
        if (int e = attn_check_tensor("sqd_attn_fwd", "k", a->k, a->k_stride, a->dtype)) return e;
        if (int e = attn_check_tensor("sqd_attn_fwd", "v", a->v, a->v_stride, a->dtype)) return e;
    }
    const Split p = plan(a);
    SQD_CHECK_ARG(p.part_floats + p.lse_floats + p.rng_floats == 0 || (a->scratch && aligned16(a->scratch)), "sqd_attn_fwd: scratch missing");
    AttnK A = attn_kargs(a);
    const hipStream_t st = (hipStream_t)a->stream;
    A.nsplit = p.nsplit, A.ntile = (int)(((int64_t)a->Sq * A.G + BM - 1) / BM), A.ndoc_tiles = p.ndoc_tiles;
    A.part_o = a->scratch, A.part_lse = a->scratch + p.part_floats;
    int2 *rng = reinterpret_cast<int2 *>(a->scratch + p.part_floats + p.lse_floats);
    A.doc_rng = rng;
    const int64_t blocks = (int64_t)A.ntile * A.nsplit * A.B * A.Hkv;
    SQD_CHECK_ARG(blocks < (1ll << 31), "sqd_attn_fwd: too many tokens");
    return for_dtype(a->dtype, [&](auto tt) {
        using T = decltype(tt);
        constexpr int KT = key_tile<T>();
        if (a->q_docs && p.ndoc_tiles) attn_doc_ranges(A.k_docs, rng, A.B, A.Sk, 1, KT, p.ndoc_tiles, st);
        auto go = [&](auto dp, auto cap, auto bias) {
            hipLaunchKernelGGL((attn_fwd_kernel<T, decltype(dp)::value, KT, decltype(cap)::value, decltype(bias)::value>), dim3((unsigned)blocks), dim3(NT),
                               0, st, A);
        };
        auto flags = [&](auto dp) {
            const bool cap = a->softcap > 0.f, bias = a->slopes != nullptr;
            if (cap && bias) go(dp, std::true_type{}, std::true_type{});
            else if (cap) go(dp, std::true_type{}, std::false_type{});
            else if (bias) go(dp, std::false_type{}, std::true_type{});
            else go(dp, std::false_type{}, std::false_type{});
        };
        switch (pad_dim(a->D)) {
            case 32: flags(std::integral_constant<int, 32>{}); break;
            case 64: flags(std::integral_constant<int, 64>{}); break;
            default: flags(std::integral_constant<int, 128>{}); break;
        }
        SQD_CHECK_LAUNCH("sqd_attn_fwd");
        if (A.nsplit > 1) {
            const int64_t units = (int64_t)A.B * A.Hkv * A.Sq * A.G * (A.D / 4);
            hipLaunchKernelGGL((attn_join_kernel<T>), dim3((unsigned)((units + NT - 1) / NT)), dim3(NT), 0, st, A);
            SQD_CHECK_LAUNCH("sqd_attn_fwd");
        }
        return SQD_OK;
    });
}
