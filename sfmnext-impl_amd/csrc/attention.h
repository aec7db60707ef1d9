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

struct AttnK {
    const void *q, *k, *v, *go;
    void *o, *gq, *gk, *gv;
    float *lse, *delta, *part_o, *part_lse;
    const float *slopes;
    const int *prefix, *q_docs, *k_docs, *k_len;
    const int2 *doc_rng;                    // per tile of the looped-over side: smallest and largest document id
    int64_t qs[3], ks[3], vs[3], gos[3];
    float scale_log2, cap_in, cap_out, cap_grad, scale;   // see Score
    int B, Sq, Sk, Hq, Hkv, G, D, causal, ntile, nsplit, ndoc_tiles;
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

// a ROWS x DP tile on its way from memory to LDS by NTH threads: 16-byte pieces in registers between load() and store()
template <typename T, int DP, int ROWS, int NTH> struct Stage {
    typedef Tile<T, DP> L;
    static constexpr int TOTAL = ROWS * L::CH, N = (TOTAL + NTH - 1) / NTH;
    u32x4 reg[N];
    // row_at(r): pointer to row r of the tile, or nullptr (zeros)
    template <typename F> __device__ __forceinline__ void load(int tid, int D, F &&row_at) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int idx = tid + n * NTH, r = idx / L::CH, c = idx % L::CH;
            u32x4 w = {0, 0, 0, 0};
            const T *p = idx < TOTAL ? row_at(r) : nullptr;
            if (p && c * L::CHE < D) w = *reinterpret_cast<const u32x4 *>(p + c * L::CHE);
            reg[n] = w;
        }
    }
    __device__ __forceinline__ void store(char *t, int tid) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int idx = tid + n * NTH;
            if (idx < TOTAL) *reinterpret_cast<u32x4 *>(t + L::at(idx / L::CH, idx % L::CH)) = reg[n];
        }
    }
};

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

// Scores in base 2: x = log2(e) (z - slope |pos - j|), z = scale q.k or c tanh(scale q.k / c).  tanh(u) = 1 - 2 / (e^{2u} + 1): one exponential and
// one reciprocal; absolute error 1e-7, i.e. 1e-7 c of a score.  cap_in = 2 log2(e) scale / c, cap_out = c log2(e).
template <bool CAP> __device__ __forceinline__ float tanh_of(float raw, float cap_in) {
    return 1.f - 2.f * __builtin_amdgcn_rcpf(exp2_hw(raw * cap_in) + 1.f);
}

// what a row may see: keys j <= lim (lengths, causal order and prefix in one number), document equal
__device__ __forceinline__ int row_limit(int pos, int len, bool causal, int prefix) { return causal ? min(max(pos, prefix - 1), len - 1) : len - 1; }

// n workgroups dealt to 8 XCDs round robin: workgroup id -> work item such that an XCD gets consecutive items (they share keys and values in
// its L2)
__device__ __forceinline__ int xcd_order(int id, int n) {
    const int x = id & 7, k = id >> 3, base = n >> 3, more = n & 7;
    return x * base + min(x, more) + k;
}
}  // namespace sqd
