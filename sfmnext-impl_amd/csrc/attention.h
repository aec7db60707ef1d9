// attention.h — what the attention kernels (attention.hip, attention_bwd.hip) share: operand fragments of the matrix instructions, the LDS tile
// layout, scores and masks.
//
// Rows.  The G = Hq / Hkv query heads that read one key head are packed behind each other: row r of (batch b, key head) is query r / G, head
// hk G + r % G.  Grouped heads then share every key / value tile, and one query token with 4 heads is 4 rows of a tile instead of 4 tiles of a row.
//
// Fragments.  Everything runs on 32x32x16 products (v_mfma_f32_32x32x16_{bf16,f16}; fp32: eight v_mfma_f32_32x32x2_f32 over the same slots, full
// precision): lane l holds 8 consecutive reduction slots 8 (l / 32) .. + 7 of row (or column) l % 32; accumulator register i of lane l is row
// (i & 3) + 8 (i >> 2) + 4 (l / 32), column l % 32.  The scores are computed so that the COLUMN is the operand a wave owns, so an accumulator's
// eight registers 8 k .. 8 k + 7 are already the operand slots of the second product if its other operand takes the reduction rows in the order
// {4 h .. 4 h + 3, 8 + 4 h .. 8 + 4 h + 3} (h = l / 32): no cross-lane traffic between the two products.
//
// LDS tiles are row-major [rows][DP] with the 16-byte pieces of a row permuted: piece c of row r sits at c ^ bitrev4(r & 15) (modulo the
// pieces of a row).  Both access patterns are then free of bank conflicts: ds_read_b128 of one piece column over 16 rows (bitrev4 is a
// permutation) and the transpose read ds_read_b64_tr_b16 of 4 rows x 64 bytes (the two low row bits go to the two HIGH piece bits, so 4
// neighbouring rows land in 4 different quarters of the 256-byte bank line).
#pragma once
#include "sqd_f16x2.h"
#include "sqd_vec.h"

namespace sqd {

struct Deal { int m, slots, share; };       // workgroups to tiles: see dealt()

struct AttnK {
    const void *q, *k, *v, *go;
    void *o, *o_low, *gq, *gk, *gv;
    float *lse, *part_o, *part_lse;
    float *row_lse, *row_delta, *row_pos, *row_slope;  // the backward's copies by packed row, padded to whole tiles (rows_padded a key head)
    int *row_lim, *row_doc;
    float *lift, *lift_max;                  // fp16 backward: see lifted()
    const float *slopes;
    const int *prefix, *q_docs, *k_docs, *k_len;
    const int2 *doc_rng;                    // per tile of the looped-over side: smallest and largest document id
    int64_t qs[3], ks[3], vs[3], gos[3];
    float scale_log2, cap_in, cap_arg, cap_out, scale;    // log2(e) scale; 2 log2(e) scale / cap, scale / cap, cap log2(e)
    unsigned g_magic;
    Deal deal;
    float unit_inv;                          // slopes are used in units of the raw score (1 / scale) or of tanh (1 / cap)
    float *part_a, *part_b;                  // the backward's parts where the looped-over side is split: [nsplit][gradient's shape]
    int B, Sq, Sk, Hq, Hkv, G, D, causal, ntile, nsplit, ndoc_tiles, rows_padded;
};

template <typename T> struct Mma;
template <> struct Mma<bf16_t> {
    typedef bf16x8 frag;
    static __device__ __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ frag pack(const float *p) {
        frag f;
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = (__bf16)p[i];
        return f;
    }
    static __device__ __forceinline__ frag rest(const float *p, frag hi) {         // what pack left
        frag f;
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = (__bf16)(p[i] - (float)hi[i]);
        return f;
    }
};
template <> struct Mma<f16_t> {
    typedef f16x8 frag;
    static __device__ __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ frag pack(const float *p) {
        frag f;
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = (_Float16)p[i];
        return f;
    }
    static __device__ __forceinline__ frag rest(const float *p, frag hi) {
        frag f;
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = (_Float16)fmaf((float)hi[i], -1.f, p[i]);       // (one instruction; exact)
        return f;
    }
};
template <> struct Mma<float> {
    struct frag { float e[8]; };
    static __device__ __forceinline__ f32x16 mma(const frag &a, const frag &b, f32x16 c) {
#pragma unroll
        for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.e[i], b.e[i], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ frag pack(const float *p) {
        frag f;
#pragma unroll
        for (int i = 0; i < 8; ++i) f.e[i] = p[i];
        return f;
    }
};

__device__ __forceinline__ int bitrev4(int r) { return ((r & 1) << 3) | ((r & 2) << 1) | ((r & 4) >> 1) | ((r & 8) >> 3); }

template <typename T, int DP> struct Tile {
    typedef typename Mma<T>::frag frag;
    static constexpr int CHE = 16 / sizeof(T);                 // elements of a 16-byte piece
    static constexpr int CH = DP / CHE;                        // pieces of a row
    static constexpr int PITCH = DP * sizeof(T);               // bytes of a row
    static constexpr int KS = DP / 16;                         // 16-slot steps over the features
    static constexpr int ROT = CH >= 16 ? 15 : CH - 1;

    static __device__ __forceinline__ int at(int row, int piece) { return row * PITCH + ((piece ^ (bitrev4(row & 15) & ROT)) << 4); }

    // features 16 ks + 8 h .. + 7 of row `row`
    static __device__ __forceinline__ frag row_frag(const char *t, int row, int ks, int h) {
        if constexpr (sizeof(T) == 2) {
            return __builtin_bit_cast(frag, *reinterpret_cast<const u32x4 *>(t + at(row, 2 * ks + h)));
        } else {
            frag f;
            const f32x4 a = *reinterpret_cast<const f32x4 *>(t + at(row, 4 * ks + 2 * h)), b = *reinterpret_cast<const f32x4 *>(t + at(row, 4 * ks + 2 * h + 1));
#pragma unroll
            for (int i = 0; i < 4; ++i) f.e[i] = a[i], f.e[4 + i] = b[i];
            return f;
        }
    }
    // the transposed operand: feature 32 db + l % 32, reduction rows kb + {4 h .. + 3, 8 + 4 h .. + 3} (kb a multiple of 16)
    static __device__ __forceinline__ frag col_frag(const char *t, int kb, int db, int lane) {
        const int h = lane >> 5;
        if constexpr (sizeof(T) == 2) {
            const int u = lane & 15, row = kb + 4 * h + (u >> 2), piece = db * 4 + 2 * ((lane >> 4) & 1) + ((u & 3) >> 1), sub = (u & 1) * 8;
            const uint2 lo = lds_read_tr16(reinterpret_cast<const unsigned short *>(t + at(row, piece) + sub));
            const uint2 hi = lds_read_tr16(reinterpret_cast<const unsigned short *>(t + at(row + 8, piece) + sub));
            const u32x4 w = {lo.x, lo.y, hi.x, hi.y};
            return __builtin_bit_cast(frag, w);
        } else {
            const int d = db * 32 + (lane & 31);
            frag f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int row = kb + 8 * (j >> 2) + 4 * h + (j & 3);
                f.e[j] = *reinterpret_cast<const float *>(t + at(row, d >> 2) + (d & 3) * 4);
            }
            return f;
        }
    }
    // features 16 ks + 8 h .. + 7 of a row in memory (D a multiple of 8); `on` false or features past D: zeros
    static __device__ __forceinline__ frag mem_frag(const T *row, int ks, int h, int D, bool on) {
        const int d = 16 * ks + 8 * h;
        if constexpr (sizeof(T) == 2) {
            u32x4 w = {0, 0, 0, 0};
            if (on && d < D) w = *reinterpret_cast<const u32x4 *>(row + d);
            return __builtin_bit_cast(frag, w);
        } else {
            f32x4 a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
            if (on && d < D) a = *reinterpret_cast<const f32x4 *>(row + d), b = *reinterpret_cast<const f32x4 *>(row + d + 4);
            frag f;
#pragma unroll
            for (int i = 0; i < 4; ++i) f.e[i] = a[i], f.e[4 + i] = b[i];
            return f;
        }
    }
};

// 16 bytes at base + off (this lane's) to LDS byte `lds` + 16 * lane, without a register in between.  The compiler does not see the load:
// dma_wait() (and a barrier, for other waves' data) comes before the LDS bytes are read.  Lanes switched off leave their 16 bytes as they are.
// (A base written by a vector instruction would want five states in between, which the compiler does not count into assembly: tests/test_kernel_waits.py
// looks for one.)
__device__ __forceinline__ void dma16(const void *base, unsigned off, unsigned lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory", "m0");
}
// (the builtin and not assembly: the compiler then knows that its own earlier loads have arrived too, and does not wait for them, and with
// them for a DMA under way, in the middle of a loop)
__device__ __forceinline__ void dma_wait() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0f70);                         // vmcnt(0)
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ unsigned lds_offset(const void *p) {
    return __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(const __attribute__((address_space(3))) char *)p);
}

// a ROWS x DP tile from memory to LDS by NTH threads.  The LDS side of a DMA is linear in the lane, so the permutation of the pieces is applied to
// the offset a lane reads.  Offsets within a tile are 32-bit and fixed (the host checks that a tile's rows span less than 2 GiB), the tile's
// base is a scalar: a tile costs one instruction a piece.  Pieces that are not loaded (rows nobody may see, features past D) keep what the buffer
// held: zeros at the start (clear_lds), later an older tile's rows, which are data of this call: finite wherever the inputs that count are.
template <typename T, int DP, int ROWS, int NTH> struct Stage {
    typedef Tile<T, DP> L;
    static constexpr int TOTAL = ROWS * L::CH, N = (TOTAL + NTH - 1) / NTH, BYTES = ROWS * L::PITCH;
    static constexpr int NO_ROW = 1 << 30;
    unsigned off[N];
    static __device__ __forceinline__ int piece_row(int n, int tid, int D) {
        const int idx = tid + n * NTH;
        return idx < TOTAL && piece_col(n, tid) < D ? idx / L::CH : NO_ROW;
    }
    static __device__ __forceinline__ int piece_col(int n, int tid) {
        const int idx = tid + n * NTH;
        return ((idx % L::CH) ^ (bitrev4((idx / L::CH) & 15) & L::ROT)) * L::CHE;
    }
    // rows `stride` elements apart
    __device__ __forceinline__ void aim(int tid, unsigned stride) {
#pragma unroll
        for (int n = 0; n < N; ++n) off[n] = ((unsigned)((tid + n * NTH) / L::CH) * stride + piece_col(n, tid)) * (unsigned)sizeof(T);
    }
    // packed rows: row r of the tile is query (rem + r) / G, head (rem + r) % G; queries s1, heads s2 elements apart
    __device__ __forceinline__ void aim_packed(int tid, int rem, int G, unsigned magic, unsigned s1, unsigned s2) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const unsigned r = rem + (tid + n * NTH) / L::CH, i = magic ? __umulhi(r, magic) : r;
            off[n] = (i * s1 + (r - i * G) * s2 + piece_col(n, tid)) * (unsigned)sizeof(T);
        }
    }
    // rows < `rows` of the tile at `base`; skip[n] < 0: not this one (with `skips`)
    __device__ __forceinline__ void load(const T *base, unsigned lds, int tid, int D, int rows, bool skips, const int (&skip)[N]) const {
        const unsigned at = lds + __builtin_amdgcn_readfirstlane(tid >> 6) * 1024;
        if (TOTAL % NTH == 0 && D == DP && rows >= ROWS && !skips) {
#pragma unroll
            for (int n = 0; n < N; ++n) dma16(base, off[n], at + n * NTH * 16);
        } else {
#pragma unroll
            for (int n = 0; n < N; ++n)
                if (piece_row(n, tid, D) < rows && (!skips || skip[n] >= 0)) dma16(base, off[n], at + n * NTH * 16);
        }
    }
};

// acc[n] += sum over the features of frag_a(n, ks) x frag_b(ks): the LDS reads of BATCH steps are in flight while the step before multiplies.  Left
// to itself the compiler reads one operand, waits for it and multiplies, and the LDS latency (some 130 cycles, against 32 of the
// product) is paid in every step; the scheduling barriers keep the batches apart.
// fp32, whose 16-feature step is eight long instructions, skips the steps past D (40 of 64 features: 3 steps of 4).
template <typename T, int NACC, int KS, int BATCH, typename FA, typename FB>
__device__ __forceinline__ void product(f32x16 (&acc)[NACC], int D, FA &&frag_a, FB &&frag_b) {
    constexpr int STEPS = NACC * KS / BATCH;
    typename Mma<T>::frag f[2][BATCH], g[2][BATCH];
    auto fetch = [&](auto st) {
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int u = decltype(st)::value * BATCH + i;
            f[decltype(st)::value & 1][i] = frag_a(u / KS, u % KS);
            g[decltype(st)::value & 1][i] = frag_b(u % KS);
        }
    };
    fetch(std::integral_constant<int, 0>{});
    static_for<STEPS>([&](auto st) {
        constexpr int S = decltype(st)::value;
        if constexpr (S + 1 < STEPS) fetch(std::integral_constant<int, S + 1>{});
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int n = (S * BATCH + i) / KS;
            if (sizeof(T) == 2 || (S * BATCH + i) % KS * 16 < D) acc[n] = Mma<T>::mma(f[S & 1][i], g[S & 1][i], acc[n]);
        }
        __builtin_amdgcn_sched_barrier(0);
    });
}
// The wait from a matrix instruction to the first other use of its result (16 bits: 8 passes, 12 states; fp32: 16 passes, 18 states), written out.  The
// compiler counts it itself, but where two ways lead to that use, one of them right behind the product, it has counted the longer one: with documents
// the token kernel then read keys 27 and 31 of a tile before the last step's product was in them.  For such places; the product() of the row kernels
// is followed by none (tests/test_kernel_waits.py looks at every way through the built kernels).
template <typename T> __device__ __forceinline__ void settle() {
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (sizeof(T) == 4) asm volatile("s_nop 15\n\ts_nop 1" ::: "memory");
    else asm volatile("s_nop 11" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
template <typename T, int KS> constexpr int batch_of() { return sizeof(T) == 4 || KS < 4 ? 2 : 4; }

// zeros over `bytes` (a multiple of 16) of LDS by NTH threads
template <int NTH> __device__ __forceinline__ void clear_lds(char *p, int bytes, int tid) {
    for (int i = tid * 16; i < bytes; i += NTH * 16) *reinterpret_cast<u32x4 *>(p + i) = u32x4{0, 0, 0, 0};
}

// the tiles of [.., end) whose documents meet [lo, hi]: 64 tiles' ranges are looked at together, one a lane, and kept as two masks
struct DocWalk {
    const int2 *rng;                        // nullptr: every tile
    int lo, hi, end, base;
    unsigned long long see, uni;
    __device__ __forceinline__ DocWalk(const int2 *r, int lo_, int hi_, int end_) : rng(r), lo(lo_), hi(hi_), end(end_), base(-64), see(0), uni(0) {}
    // first tile >= t, `end` if none; one_doc: the tile and [lo, hi] are one and the same document
    __device__ __forceinline__ int next(int t, bool &one_doc) {
        one_doc = true;
        if (!rng) return min(t, end);
        while (t < end) {
            if (t - base >= 64) {
                base = t & ~63;
                const int u = base + (int)__lane_id();
                int2 r = make_int2(0x7fffffff, -1);
                if (u < end) r = rng[u];
                see = __ballot(r.y >= lo && r.x <= hi);
                uni = __ballot(lo == hi && r.x == lo && r.y == lo);
            }
            const unsigned long long m = see >> (t - base);
            if (m) {
                t += __builtin_ctzll(m);
                one_doc = (uni >> (t - base)) & 1;
                return t;
            }
            t = base + 64;
        }
        return end;
    }
};

// R / G by a multiplication (R G < 2^32, checked on the host); magic = ceil(2^32 / G), 0 for G = 1
__device__ __forceinline__ int div_g(int R, unsigned magic) { return magic ? (int)__umulhi((unsigned)R, magic) : R; }

// the larger / sum of the two half-waves' values, in both halves
__device__ __forceinline__ float half_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// The forms of a capped score, chosen on the host (cap_form) and compiled apart.  CAP_SHORT: tanh u = 1 - 2 / (e^{2u} + 1), one exponential and one
// reciprocal, absolute error 4 2^-24, i.e. that times the cap in the score.  Twice that (a score and the row's largest) stays below 2^-14 of a
// probability, an eighth of half a step of fp16, up to a cap of 128: 16-bit types take it there.  CAP_FULL: the library's tanh, whose error is
// relative.  fp32 always takes it, and 16-bit types past 128 (a cap of 10^4 leaves 2.4e-3 of a score in the short form, one of 10^8 no score at all).
enum { CAP_NONE = 0, CAP_SHORT = 1, CAP_FULL = 2 };
inline int cap_form(float softcap, int dtype) { return softcap == 0.f ? CAP_NONE : dtype != SQD_F32 && softcap <= 128.f ? CAP_SHORT : CAP_FULL; }
// f(form, bias) as compile-time constants
template <typename T, typename F> inline void for_scores(int cap, bool bias, F &&f) {
    auto form = [&](auto c) {
        if (bias) f(c, std::true_type{});
        else f(c, std::false_type{});
    };
    if (cap == CAP_NONE) form(std::integral_constant<int, CAP_NONE>{});
    else if (cap == CAP_FULL) form(std::integral_constant<int, CAP_FULL>{});
    else if constexpr (sizeof(T) == 2) form(std::integral_constant<int, CAP_SHORT>{});
}
// tanh of a capped score (raw: the product before the scale)
template <int CAP> __device__ __forceinline__ float tanh_of(float raw, const AttnK &A) {
    if constexpr (CAP == CAP_FULL) return tanhf(raw * A.cap_arg);
    else return fmaf(-2.f, __builtin_amdgcn_rcpf(exp2_hw(raw * A.cap_in) + 1.f), 1.f);
}

// fp16 keeps 11 bits down to 2^-14 only, and P and dS are far smaller: 1 / (keys of a row), times the incoming gradient.  They are packed multiplied
// by powers of two that the results are divided by in fp32: P by 2^P_LIFT, dS by the largest 2^k that keeps
// |P (dP - delta)| <= |go_i| |v_j| + |delta_i| below 2^15 for each pair of a batch row's key head (attn_rows_kernel takes the three maxima).
template <typename T> constexpr bool lifted() { return std::is_same<T, f16_t>::value; }
constexpr float P_LIFT = 14.f, P_SCALE = 16384.f;               // P_SCALE = 2^P_LIFT

// what a row may see: keys j <= lim (lengths, causal order and prefix in one number), document equal
__device__ __forceinline__ int row_limit(int pos, int len, bool causal, int prefix) { return causal ? min(max(pos, prefix - 1), len - 1) : len - 1; }

// what one lane knows of its row
struct RowOf {
    int i, g, pos, qd, lim;
    bool on;
};
__device__ __forceinline__ RowOf row_of(const AttnK &A, int b, int R, int RT, int len, int prefix) {
    RowOf r;
    r.on = R < RT;
    r.i = r.on ? div_g(R, A.g_magic) : A.Sq - 1;
    r.g = r.on ? R - r.i * A.G : 0;
    r.pos = r.i + len - A.Sq;
    r.qd = -2;
    if (A.q_docs && r.on) r.qd = max(A.q_docs[(int64_t)b * A.Sq + r.i], -1);
    if (r.qd == -1) r.qd = -2;
    r.lim = r.on && (!A.q_docs || r.qd >= 0) ? row_limit(r.pos, len, A.causal, prefix) : -1;
    return r;
}

// Workgroups are dealt to the 8 XCDs round robin; the ones that share keys and values (a group: one batch row's key head) belong on one XCD and its
// L2.  With a number of groups that 8 does not divide a group is shared by m = 8 / gcd(8, groups) XCDs, its tiles dealt in turn: in causal
// order the tiles' work grows along the group, and consecutive halves would be as 1 to 3 (8192 tokens, 4 groups: 410 us that way).
// id -> group and tile, the last tile first; false: no such tile.
inline Deal deal(int groups, int tiles) {
    const int g = groups % 8 == 0 ? 8 : groups % 4 == 0 ? 4 : groups % 2 == 0 ? 2 : 1;
    Deal d;
    d.m = 8 / g;
    d.slots = (tiles + d.m - 1) / d.m;
    d.share = groups / g;                   // sub-groups an XCD takes
    return d;
}
inline int64_t deal_blocks(const Deal &d) { return (int64_t)8 * d.share * d.slots; }
__device__ __forceinline__ bool dealt(const Deal &d, int id, int tiles, int &group, int &tile) {
    const int x = id & 7, k = id >> 3, local = k / d.slots, j = k - local * d.slots, sub = x * d.share + local;
    group = sub / d.m;
    tile = j * d.m + sub - group * d.m;
    return tile < tiles;
}
}  // namespace sqd
