// attention.hip — attention forward for packed / causal / prefix / cached tokens with capped scores and a bias by distance (include/sqd.h
// section 22).  o = softmax(z) v over the keys a row may see, one pass over the keys with a running maximum and sum (fp32, base 2).
//
// Four waves of 32 rows share the key tiles (64 keys; 32 in fp32), two buffers, the next tile on its way by DMA while one is used.  A row tile walks
// only the key tiles its rows may see: lengths, causal order and prefix end the walk, document ranges skip tiles; the mask itself is applied only in
// tiles that some row sees in part.
// Measured (library product of 8192^3 on the same card: 1218 bf16 / 1176 fp16 / 153 fp32 TFLOP/s): 8192 causal fp16 tokens behind a prefix of 1280, 16 + 4
// heads of 128: 321 .. 327 us = 870 TFLOP/s of what the masks leave, the matrix pipe 0.50 and the vector pipe 0.54 of the time busy; 2 x 3840 bf16 in 3
// documents, capped: 134 us = 490 (the cap's exponential and reciprocal are vector work: vector 0.56, matrix 0.23); 12 x 480, 12 heads of 64, bf16,
// distance bias: 32 us (0.51, 0.17); 2 x 1281 fp32, 8 heads of 40, causal: 54 us (matrix 0.64).  The products and the softmax of a wave follow each other,
// which is what keeps either pipe from being full.  No LDS bank conflicts in the row kernel; the token kernel's join has some (0.31 of its few LDS cycles:
// rows of 512 bytes).
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

// four neighbouring features of the output, and what their rounding left (o_low: the backward's delta wants o to more bits than o has)
template <typename T> __device__ __forceinline__ void store_out(const AttnK &A, int64_t at, const float (&v)[4]) {
    store_f32<T, 4>((T *)A.o + at, v);
    if (sizeof(T) == 2 && A.o_low) {
        float r[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = v[e] - to_f32(from_f32<T>(v[e]));
        store_f32<T, 4>((T *)A.o_low + at, r);
    }
}

// The scores of one tile (x: raw products, NB blocks of 32 keys by the wave's 32 rows), the running maximum and sum, and the second product.
template <typename T, int DP, int NB, int CAP, bool BIAS> struct Softmax {
    typedef Tile<T, DP> L;
    static constexpr int DB = DP / 32;
    // fp16: P below 2^-14 of the row's largest would lose bits and below 2^-25 all of them, however many keys there are: it is packed times 2^P_LIFT.
    // o and l hold that factor, their quotient does not.  m is a multiple of 2^-18 then, so that m - P_LIFT is exact (up to 50): lse keeps all its bits,
    // which the backward's P = 1 of a single key wants
    static constexpr float UP = lifted<T>() ? P_LIFT : 0.f, DOWN = lifted<T>() ? 1.f / P_SCALE : 1.f;
    static __device__ __forceinline__ float lse(float m, float l) {
        const float d = l * DOWN - 1.f;     // next to one, where a single key's sum is, the hardware's logarithm is short of bits
                                            // (up to 2^-12 the second term, d^2 / 2, is below 2^-25)
        return m + (lifted<T>() && fabsf(d) < 1.f / 4096.f ? d * 1.44269504f : __builtin_amdgcn_logf(l * DOWN));
    }
    f32x16 o[DB];
    float m, l;
    __device__ __forceinline__ Softmax() : m(-INFINITY), l(0.f) {
#pragma unroll
        for (int db = 0; db < DB; ++db) o[db] = f32x16{};
    }
    // j0: first key; lim, qd: the row's limit and document; ld: the tile's documents (docs); part: some row does not see the whole tile
    __device__ __forceinline__ void tile(f32x16 (&x)[NB], const AttnK &A, const char *lv, const int *ld, bool docs, bool part, int j0, int pos, int lim, int qd,
                                         float slope, int lane) {
        const int h = lane >> 5;
        // scores in units of c = log2(e) scale, or of c = log2(e) cap behind tanh: c goes into the exponent's fma
        const float c = CAP ? A.cap_out : A.scale_log2, d0 = (float)(pos - j0 - 4 * h);
        if (CAP || BIAS) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    if (CAP) x[nb][r] = tanh_of<CAP>(x[nb][r], A);
                    if (BIAS) x[nb][r] = fmaf(-slope, fabsf(d0 - (float)(nb * 32 + (r & 3) + 8 * (r >> 2))), x[nb][r]);
                }
        }
        if (part) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) {
                    const int j4 = nb * 32 + 8 * r4 + 4 * h;
                    int4 kd = make_int4(qd, qd, qd, qd);
                    if (docs) kd = *reinterpret_cast<const int4 *>(ld + j4);
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
        mx = half_max(mx) * c;
        if (lifted<T>() && fabsf(mx) < 64.f) mx = rintf(mx * 262144.f) * (1.f / 262144.f);
        const float mn = fmaxf(m, mx);
        if (__builtin_expect(__any(mn > m), 0)) {              // rare once the maximum has settled
            const float alpha = exp2_hw(m - (mn == -INFINITY ? 0.f : mn));
            l *= alpha;
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
            m = mn;
        }
        const float base = (m == -INFINITY ? 0.f : m) - UP;
        // 16 keys at a time: their values' operands are read while the step before multiplies, and the exponentials of a step run under its products
        typename L::frag vf[2][DB];
#pragma unroll
        for (int db = 0; db < DB; ++db) vf[0][db] = L::col_frag(lv, 0, db, lane);
        static_for<2 * NB>([&](auto step) {
            constexpr int K = decltype(step)::value;
            float p[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                p[r] = exp2_hw(fmaf(x[K / 2][8 * (K & 1) + r], c, -base));
                l += p[r];
            }
            // P is rounded to the values' type for the second product (half a step of that type, relative); the sum keeps the unrounded P
            const typename L::frag pf = Mma<T>::pack(p);
            if constexpr (K + 1 < 2 * NB)
#pragma unroll
                for (int db = 0; db < DB; ++db) vf[(K + 1) & 1][db] = L::col_frag(lv, (K + 1) * 16, db, lane);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int db = 0; db < DB; ++db) o[db] = Mma<T>::mma(vf[K & 1][db], pf, o[db]);
        });
    }
};

template <typename T, int DP, int KT, int CAP, bool BIAS>
__global__ __launch_bounds__(NT, DP * sizeof(T) > 256 ? 1 : DP * sizeof(T) > 128 ? 2 : 3) void attn_fwd_kernel(AttnK A) {
    typedef Tile<T, DP> L;
    typedef typename L::frag frag;
    typedef Stage<T, DP, KT, NT> S;
    constexpr int NB = KT / 32, DB = DP / 32;
    __shared__ __align__(16) char lk[2][S::BYTES], lv[2][S::BYTES];
    __shared__ __align__(16) int ld[2][KT];
    __shared__ int wq[8];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    int bh, w;
    if (!dealt(A.deal, blockIdx.x, A.ntile * A.nsplit, bh, w)) return;
    const int split = w % A.nsplit, tile = A.ntile - 1 - w / A.nsplit, hk = bh % A.Hkv, b = bh / A.Hkv;        // the longest causal rows first
    const int RT = A.Sq * A.G, row0 = tile * BM;
    const int len = A.k_len ? min(max(A.k_len[b], 0), A.Sk) : A.Sk;
    const int prefix = A.prefix ? max(A.prefix[b], 0) : 0;
    const int R = row0 + wave * 32 + (lane & 31);               // this lane's row (both half-waves hold the same 32)
    const RowOf row = row_of(A, b, R, RT, len, prefix);
    clear_lds<NT>(lk[0], 2 * S::BYTES, tid);
    clear_lds<NT>(lv[0], 2 * S::BYTES, tid);

    // keys any row of the workgroup may see
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
    const int nt_all = (kend + KT - 1) / KT, per = (nt_all + A.nsplit - 1) / A.nsplit;
    const int t0 = min(nt_all, split * per), t1 = min(nt_all, t0 + per);
    DocWalk walk(A.q_docs ? A.doc_rng + (int64_t)b * A.ndoc_tiles : nullptr, dlo, dhi, t1);

    frag qf[L::KS];
    const T *qrow = (const T *)A.q + b * A.qs[0] + (int64_t)row.i * A.qs[1] + (int64_t)(hk * A.G + row.g) * A.qs[2];
#pragma unroll
    for (int ks = 0; ks < L::KS; ++ks) qf[ks] = L::mem_frag(qrow, ks, h, A.D, row.on);

    const T *kbase = (const T *)A.k + b * A.ks[0] + hk * A.ks[2], *vbase = (const T *)A.v + b * A.vs[0] + hk * A.vs[2];
    const int *kdoc = A.k_docs ? A.k_docs + (int64_t)b * A.Sk : nullptr;
    S sk, sv;
    sk.aim(tid, (unsigned)A.ks[1]);
    sv.aim(tid, (unsigned)A.vs[1]);
    const unsigned ok = lds_offset(lk[0]), ov = lds_offset(lv[0]);
    // padding keys (a negative document) are not loaded: their documents are read a tile ahead of the DMA that goes by them
    int pd[S::N], sd = -1;
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
    Softmax<T, DP, NB, CAP, BIAS> sm;
    bool u, un;
    int t = walk.next(t0, u);
    peek(t);
    if (t < t1) fetch(t, 0);
    int tn = walk.next(t + 1, un);
    peek(tn);
    dma_wait();
    __syncthreads();
    // the two buffers as two copies of the loop body: LDS addresses are then constants of a lane (40 of 295 vector instructions a tile less)
    auto step = [&](auto buffer) __attribute__((always_inline)) {
        constexpr int s = decltype(buffer)::value;
        if (tn < t1) fetch(tn, s ^ 1);
        bool u2 = true;
        const int t2 = walk.next(tn + 1, u2);
        peek(t2);
        f32x16 x[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) x[nb] = f32x16{};
        product<T, NB, L::KS, batch_of<T, L::KS>()>(
            x, A.D, [&](int nb, int ks) { return L::row_frag(lk[s], nb * 32 + (lane & 31), ks, h); }, [&](int ks) { return qf[ks]; });
        // the mask, where a row of the wave does not see the whole tile
        const bool part = !u || __any(row.lim < t * KT + KT - 1);
        sm.tile(x, A, lv[s], ld[s], kdoc != nullptr, part, t * KT, row.pos, row.lim, row.qd, slope, lane);
        dma_wait();
        __syncthreads();
        t = tn, u = un, tn = t2, un = u2;
    };
    while (t < t1) {
        step(std::integral_constant<int, 0>{});
        if (t >= t1) break;
        step(std::integral_constant<int, 1>{});
    }

    const float l = half_sum(sm.l), inv = l > 0.f || l != l ? 1.f / l : 0.f;
    if (!row.on) return;
    const int64_t at = (int64_t)bh * RT + R;
    if (A.nsplit > 1) {
        float *po = A.part_o + ((int64_t)split * A.B * A.Hkv * RT + at) * A.D;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                const int d = db * 32 + 8 * r4 + 4 * h;
                const float v[4] = {sm.o[db][4 * r4] * inv, sm.o[db][4 * r4 + 1] * inv, sm.o[db][4 * r4 + 2] * inv, sm.o[db][4 * r4 + 3] * inv};
                if (d < A.D) store_f32<float, 4>(po + d, v);
            }
        if (h == 0) A.part_lse[(int64_t)split * A.B * A.Hkv * RT + at] = l == 0.f ? -INFINITY : sm.lse(sm.m, l);
        return;
    }
    const int64_t out_at = (((int64_t)b * A.Sq + row.i) * A.Hq + hk * A.G + row.g) * A.D;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            const int d = db * 32 + 8 * r4 + 4 * h;
            const float v[4] = {sm.o[db][4 * r4] * inv, sm.o[db][4 * r4 + 1] * inv, sm.o[db][4 * r4 + 2] * inv, sm.o[db][4 * r4 + 3] * inv};
            if (d < A.D) store_out<T>(A, out_at + d, v);
        }
    if (A.lse && h == 0) A.lse[at] = l == 0.f ? INFINITY : sm.lse(sm.m, l);
}

// Few rows (Sq G <= 32: one or some tokens against a cache).  Bandwidth bound, so what counts is bytes in flight: every wave takes 32 keys of its
// own at a time, its K and V rows go by DMA into two private buffers, and no wave waits for another until the end, where the waves' maxima,
// sums and outputs are joined through LDS.  Wave w of split s takes the key tiles s * per + w, + NW, ...
// Measured: 16 tokens, 32 + 8 heads of 128 bf16, caches of 4351 to 8191 keys (411 MB): 88 us = 4.7 TB/s, and 5 us for the join of the two parts.
template <typename T, int DP> constexpr int token_waves() { return sizeof(T) == 4 && DP == 128 ? 2 : 4; }       // 64 KB of buffers a wave in fp32
template <typename T, int DP, int NW, int CAP, bool BIAS>
__global__ __launch_bounds__(64 * NW) void attn_token_kernel(AttnK A) {
    typedef Tile<T, DP> L;
    typedef typename L::frag frag;
    typedef Stage<T, DP, 32, 64> S;
    constexpr int DB = DP / 32;
    static_assert(4 * S::BYTES >= 32 * DP * 4, "the buffers of a wave hold its 32 output rows in fp32");
    __shared__ __align__(16) char buf[NW][4 * S::BYTES];        // K, V, K, V
    __shared__ __align__(16) int ld[NW][32];
    __shared__ float wm[NW][32], wl[NW][32];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    // no two workgroups share keys: the splits of a row of the batch, whose lengths differ, go round the XCDs
    const int groups = A.B * A.Hkv, split = blockIdx.x / groups, bh = blockIdx.x - split * groups, hk = bh % A.Hkv, b = bh / A.Hkv;
    const int RT = A.Sq * A.G, R = lane & 31;
    const int len = A.k_len ? min(max(A.k_len[b], 0), A.Sk) : A.Sk;
    const int prefix = A.prefix ? max(A.prefix[b], 0) : 0;
    const RowOf row = row_of(A, b, R, RT, len, prefix);
    clear_lds<64>(buf[wave], 4 * S::BYTES, lane);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    // (causal: the last query sees every key; keys of other documents are hidden pair by pair)
    const int nt_all = (len + 31) / 32, per = ((nt_all + A.nsplit - 1) / A.nsplit + NW - 1) / NW * NW;
    const int t0 = min(nt_all, split * per), t1 = min(nt_all, t0 + per);

    frag qf[L::KS];
    const T *qrow = (const T *)A.q + b * A.qs[0] + (int64_t)row.i * A.qs[1] + (int64_t)(hk * A.G + row.g) * A.qs[2];
#pragma unroll
    for (int ks = 0; ks < L::KS; ++ks) qf[ks] = L::mem_frag(qrow, ks, h, A.D, row.on);
    const T *kbase = (const T *)A.k + b * A.ks[0] + hk * A.ks[2], *vbase = (const T *)A.v + b * A.vs[0] + hk * A.vs[2];
    const int *kdoc = A.k_docs ? A.k_docs + (int64_t)b * A.Sk : nullptr;
    S sk, sv;
    sk.aim(lane, (unsigned)A.ks[1]);
    sv.aim(lane, (unsigned)A.vs[1]);
    const unsigned o0 = lds_offset(buf[wave]);
    auto fetch = [&](int t, int s) {
        const int j0 = t * 32;
        int pd[S::N];
        if (kdoc)
#pragma unroll
            for (int n = 0; n < S::N; ++n) {
                const int r = S::piece_row(n, lane, A.D);
                pd[n] = r < len - j0 ? kdoc[j0 + r] : -1;
            }
        sk.load(kbase + (int64_t)j0 * A.ks[1], o0 + s * 2 * S::BYTES, lane, A.D, len - j0, kdoc != nullptr, pd);
        sv.load(vbase + (int64_t)j0 * A.vs[1], o0 + (s * 2 + 1) * S::BYTES, lane, A.D, len - j0, kdoc != nullptr, pd);
    };
    const float slope = BIAS && row.on ? A.slopes[hk * A.G + row.g] * A.unit_inv : 0.f;
    Softmax<T, DP, 1, CAP, BIAS> sm;
    int t = t0 + wave, s = 0;
    if (t < t1) fetch(t, 0);
    while (t < t1) {
        dma_wait();
        if (t + NW < t1) fetch(t + NW, s ^ 1);
        const int j0 = t * 32;
        if (kdoc && lane < 32) ld[wave][lane] = j0 + lane < len ? kdoc[j0 + lane] : -1;
        const char *lk = buf[wave] + s * 2 * S::BYTES, *lv = lk + S::BYTES;
        f32x16 x[1] = {f32x16{}};
        product<T, 1, L::KS, batch_of<T, L::KS>()>(
            x, A.D, [&](int, int ks) { return L::row_frag(lk, lane & 31, ks, h); }, [&](int ks) { return qf[ks]; });
        settle<T>();
        const bool part = kdoc != nullptr || __any(row.lim < j0 + 31);
        sm.tile(x, A, lv, ld[wave], kdoc != nullptr, part, j0, row.pos, row.lim, row.qd, slope, lane);
        t += NW;
        s ^= 1;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // this buffer is read before the next turn's DMA overwrites it
    }
    // join the waves: the row's common maximum, then the weighted sums
    const float l = half_sum(sm.l);
    if (h == 0) wm[wave][R] = l == 0.f ? -INFINITY : sm.m, wl[wave][R] = l;
    __syncthreads();
    float mx = wm[0][R];
#pragma unroll
    for (int k = 1; k < NW; ++k) mx = fmaxf(mx, wm[k][R]);
    const float base = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < NW; ++k) sum += wl[k][R] * exp2_hw(wm[k][R] - base);
    const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f, mine = (l == 0.f ? 0.f : exp2_hw(sm.m - base)) * inv;
    float *po = reinterpret_cast<float *>(buf[wave]);           // [32][DP]
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            const f32x4 v = {sm.o[db][4 * r4] * mine, sm.o[db][4 * r4 + 1] * mine, sm.o[db][4 * r4 + 2] * mine, sm.o[db][4 * r4 + 3] * mine};
            *reinterpret_cast<f32x4 *>(po + R * DP + db * 32 + 8 * r4 + 4 * h) = v;
        }
    __syncthreads();
    const int64_t rows = (int64_t)A.B * A.Hkv * RT, at0 = (int64_t)bh * RT;
    for (int u = tid; u < RT * (DP / 4); u += 64 * NW) {
        const int r = u / (DP / 4), d = u % (DP / 4) * 4;
        if (d >= A.D) continue;
        f32x4 a = *reinterpret_cast<const f32x4 *>(reinterpret_cast<const float *>(buf[0]) + r * DP + d);
#pragma unroll
        for (int k = 1; k < NW; ++k) a += *reinterpret_cast<const f32x4 *>(reinterpret_cast<const float *>(buf[k]) + r * DP + d);
        const float v[4] = {a[0], a[1], a[2], a[3]};
        if (A.nsplit > 1) {
            store_f32<float, 4>(A.part_o + ((int64_t)split * rows + at0 + r) * A.D + d, v);
        } else {
            const int i = div_g(r, A.g_magic), g = r - i * A.G;
            store_out<T>(A, (((int64_t)b * A.Sq + i) * A.Hq + hk * A.G + g) * A.D + d, v);
        }
    }
    if (tid < RT) {                                             // tid < 32: lane = row
        if (A.nsplit > 1) A.part_lse[(int64_t)split * rows + at0 + R] = sum == 0.f ? -INFINITY : sm.lse(mx, sum);
        else if (A.lse) A.lse[at0 + R] = sum == 0.f ? INFINITY : sm.lse(mx, sum);
    }
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
    const int R = (int)(at - bh * RT), i = div_g(R, A.g_magic), g = R - i * A.G, hk = (int)(bh % A.Hkv);
    store_out<T>(A, (((bh / A.Hkv) * A.Sq + i) * A.Hq + hk * A.G + g) * A.D + d, a);
    if (A.lse && d == 0) A.lse[at] = sum == 0.f ? INFINITY : mx + __builtin_amdgcn_logf(sum);
}

template <typename T> constexpr int key_tile() { return sizeof(T) == 4 ? 32 : 64; }
int pad_dim(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }

struct Split { bool token; int nsplit, ndoc_tiles; int64_t part_floats, lse_floats, rng_floats; };
Split plan(const sqd_attn_args *a) {
    const int G = a->Hq / a->Hkv;
    const int64_t rows = (int64_t)a->Sq * G;
    Split p{};
    p.token = rows <= 32;
    const int KT = p.token ? 32 : a->dtype == SQD_F32 ? 32 : 64;
    const int64_t groups = (int64_t)a->B * a->Hkv * (p.token ? 1 : (rows + BM - 1) / BM);
    // split the keys while CUs would idle, down to 256 keys for each: two workgroups of the row kernel fit a CU; of the token kernel as many as its
    // buffers leave room for (one at 128 features of 16 bits: 512 instead of 256 workgroups cost 95 against 87 us on 16 x 8 key heads of 8191)
    const int bytes = pad_dim(a->D) * (a->dtype == SQD_F32 ? 4 : 2), want = p.token ? 256 * (bytes >= 256 ? 1 : 256 / bytes) : 512;
    const int tiles = (a->Sk + KT - 1) / KT;
    int64_t n = groups ? want / groups : 1;
    n = n > a->Sk / 256 ? a->Sk / 256 : n;
    p.nsplit = (int)(n < 1 ? 1 : n > 64 ? 64 : n);
    p.ndoc_tiles = a->q_docs && !p.token ? tiles : 0;
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
    SQD_CHECK_ARG(a->Sk < (1 << 24) && (int64_t)a->Sq * (a->Hq / a->Hkv) < (1 << 30) &&
                      (int64_t)a->Sq * (a->Hq / a->Hkv) * (a->Hq / a->Hkv) < (1ll << 31) && (int64_t)a->B * a->Hkv < (1 << 24) && a->B < 65536 && a->Hkv < 65536, "%s: too many tokens", who);
    SQD_CHECK_ARG(a->scale > 1e-30f && a->scale < 1e30f && a->softcap >= 0.f && a->softcap < 1e30f && (a->softcap == 0.f || a->softcap > 1e-30f), "%s: scale %g, cap %g", who, (double)a->scale, (double)a->softcap);
    SQD_CHECK_ARG(a->dtype >= SQD_F32 && a->dtype <= SQD_F16, "%s: element type %d", who, a->dtype);
    SQD_CHECK_ARG(!a->prefix || a->causal, "%s: a prefix needs the causal order", who);
    SQD_CHECK_ARG(!a->q_docs == !a->k_docs, "%s: documents of queries and keys come together", who);
    return SQD_OK;
}
// a tile of rows (up to 128 tokens, or 64 packed rows of G heads) is addressed by 32-bit offsets
int attn_check_tensor(const char *who, const char *name, const void *p, const int64_t *stride, int heads, int dtype) {
    const int V = dtype == SQD_F32 ? 4 : 8;
    SQD_CHECK_ARG(stride[1] >= 0 && stride[1] < (1 << 22) && stride[2] >= 0 && stride[2] * heads < (1 << 28), "%s: token / head strides of %s: %lld, %lld", who, name,
                  (long long)stride[1], (long long)stride[2]);
    SQD_CHECK_ARG(p && aligned16(p) && stride[0] % V == 0 && stride[1] % V == 0 && stride[2] % V == 0, "%s: %s must be 16-byte aligned, its strides too", who, name);
    return SQD_OK;
}
AttnK attn_kargs(const sqd_attn_args *a) {
    AttnK A{};
    A.q = a->q, A.k = a->k, A.v = a->v, A.go = a->go, A.o = a->o, A.o_low = a->o_low, A.gq = a->gq, A.gk = a->gk, A.gv = a->gv, A.lse = a->lse;
    A.slopes = a->slopes, A.prefix = a->prefix, A.q_docs = a->q_docs, A.k_docs = a->k_docs, A.k_len = a->k_len;
    for (int i = 0; i < 3; ++i) A.qs[i] = a->q_stride[i], A.ks[i] = a->k_stride[i], A.vs[i] = a->v_stride[i], A.gos[i] = a->go_stride[i];
    constexpr double LOG2E = 1.44269504088896340736;
    A.scale = a->scale;
    A.scale_log2 = (float)(a->scale * LOG2E);
    A.unit_inv = (float)(1.0 / (a->softcap > 0.f ? a->softcap : a->scale));
    if (a->softcap > 0.f) A.cap_in = (float)(2.0 * LOG2E * a->scale / a->softcap), A.cap_arg = (float)((double)a->scale / a->softcap), A.cap_out = (float)(a->softcap * LOG2E);
    A.B = a->B, A.Sq = a->Sq, A.Sk = a->Sk, A.Hq = a->Hq, A.Hkv = a->Hkv, A.G = a->Hq / a->Hkv, A.D = a->D, A.causal = a->causal;
    A.g_magic = A.G == 1 ? 0u : (unsigned)(((1ull << 32) + A.G - 1) / A.G);
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
    if (int e = attn_check_tensor("sqd_attn_fwd", "q", a->q, a->q_stride, a->Hq, a->dtype)) return e;
    if (a->Sk) {
        if (int e = attn_check_tensor("sqd_attn_fwd", "k", a->k, a->k_stride, a->Hkv, a->dtype)) return e;
        if (int e = attn_check_tensor("sqd_attn_fwd", "v", a->v, a->v_stride, a->Hkv, a->dtype)) return e;
    }
    const Split p = plan(a);
    SQD_CHECK_ARG(p.part_floats + p.lse_floats + p.rng_floats == 0 || (a->scratch && aligned16(a->scratch)), "sqd_attn_fwd: scratch missing");
    AttnK A = attn_kargs(a);
    const hipStream_t st = (hipStream_t)a->stream;
    A.nsplit = p.nsplit, A.ntile = (int)(((int64_t)a->Sq * A.G + BM - 1) / BM), A.ndoc_tiles = p.ndoc_tiles;
    A.part_o = a->scratch, A.part_lse = a->scratch + p.part_floats;
    int2 *rng = reinterpret_cast<int2 *>(a->scratch + p.part_floats + p.lse_floats);
    A.doc_rng = rng;
    const int64_t tiles = (int64_t)A.ntile * A.nsplit;
    SQD_CHECK_ARG(tiles < (1 << 24), "sqd_attn_fwd: too many tokens");
    A.deal = deal(A.B * A.Hkv, (int)tiles);
    const int64_t blocks = p.token ? tiles * A.B * A.Hkv : deal_blocks(A.deal);
    SQD_CHECK_ARG(blocks <= max_blocks(NT), "sqd_attn_fwd: too many tokens");
    return for_dtype(a->dtype, [&](auto tt) {
        using T = decltype(tt);
        constexpr int KT = key_tile<T>();
        if (p.ndoc_tiles) attn_doc_ranges(A.k_docs, rng, A.B, A.Sk, 1, KT, p.ndoc_tiles, st);
        auto go = [&](auto dp, auto cap, auto bias) {
            if (p.token)
                hipLaunchKernelGGL((attn_token_kernel<T, decltype(dp)::value, token_waves<T, decltype(dp)::value>(), decltype(cap)::value, decltype(bias)::value>),
                                   dim3((unsigned)blocks), dim3(64 * token_waves<T, decltype(dp)::value>()), 0, st, A);
            else
                hipLaunchKernelGGL((attn_fwd_kernel<T, decltype(dp)::value, KT, decltype(cap)::value, decltype(bias)::value>), dim3((unsigned)blocks), dim3(NT),
                               0, st, A);
        };
        auto flags = [&](auto dp) { for_scores<T>(cap_form(a->softcap, a->dtype), a->slopes != nullptr, [&](auto cap, auto bias) { go(dp, cap, bias); }); };
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
