// rotary.hip — rotary positions over several axes (time, row, column) for queries and keys (include/sqd.h section 21).
//
// P pairs of a head's D features turn by angle_p = position[axis(p)] * freq_p; the pairs are (p, p + P) or, interleaved, (2p, 2p + 1), the
// trailing D - 2P features pass unchanged:      (a, b) -> (a cos - b sin, b cos + a sin).      The backward is the turn by -angle_p.
//
// Angles: a position of 10^6 times a frequency of 1 has lost its fraction in fp32 (one unit in the last place is 0.06 rad), so the product is
// taken in fp64, reduced to turns in [-1/2, 1/2] there, and only the fraction goes to sincospi in fp32 (absolute error < 2^-23 of a turn).  A
// workgroup takes a few tokens, computes their P angles once into LDS and applies them to all query and key heads: the trigonometry is
// 1 / (Hq + Hk) of a per-element evaluation and the kernel stays HBM bound (every element read and written once, 16-byte pieces).  Queries and
// keys go in one launch.
// Measured: 40960 tokens, 16 + 4 heads of 128 bf16, 3 axes: 420 MB in 88 us = 4.8 TB/s (a plain copy: 5.0); 12 tokens 4.9 us, all latency.
#include "sqd_vec.h"

namespace {
using namespace sqd;

constexpr int NT = 256, MAX_AXES = 4, MAX_TOKENS = 16;

struct RotaryArgs {
    const void *x[2];                  // queries, keys
    void *y[2];                        // dense [B,S,H,D]
    int64_t xb[2], xs[2], xh[2];       // element strides of batch, token, head
    int heads[2];
    const void *pos;                   // [S,A] or [B,S,A]
    int64_t pos_b;
    const double *freq;                // [P] radians per unit of position
    int axis_end[MAX_AXES];            // pairs below axis_end[a] (and not below axis_end[a-1]) belong to axis a
    int S, D, P, A, tokens;            // tokens per workgroup
    int64_t BS, first;                 // first: the launch's first token
    float sign;
};

template <typename T, typename I, int VEC, bool PAIRED>
__global__ __launch_bounds__(NT) void rotary_kernel(RotaryArgs R) {
    extern __shared__ float2 cs[];                              // [tokens][P] cos, sin
    __shared__ int64_t src_at[2][MAX_TOKENS];                   // a token's first element in queries / keys
    const int64_t t0 = R.first + (int64_t)blockIdx.x * R.tokens;
    const int nt = (int)min((int64_t)R.tokens, R.BS - t0);
    if (threadIdx.x < 2 * MAX_TOKENS && (int)(threadIdx.x % MAX_TOKENS) < nt) {
        const int w = threadIdx.x / MAX_TOKENS, t = threadIdx.x % MAX_TOKENS;
        const int64_t bs = t0 + t, b = bs / R.S, s = bs - b * R.S;
        src_at[w][t] = b * R.xb[w] + s * R.xs[w];
    }
    for (int u = threadIdx.x; u < nt * R.P; u += NT) {
        const int t = u / R.P, p = u - t * R.P;
        int a = 0;
        while (a + 1 < R.A && p >= R.axis_end[a]) ++a;
        const int64_t bs = t0 + t, b = bs / R.S, s = bs - b * R.S;
        const double at = (double)reinterpret_cast<const I *>(R.pos)[b * R.pos_b + s * R.A + a];
        double turns = at * R.freq[p] * 0.15915494309189533577;                 // 1 / (2 pi)
        turns -= rint(turns);
        float sn, c;
        sincospif(2.f * (float)turns, &sn, &c);
        cs[u] = make_float2(c, R.sign * sn);
    }
    __syncthreads();
    // units of one head: pieces of VEC pairs first, then pieces of VEC features that pass through.  A thread keeps its unit (its head and
    // piece: two divisions a call) and walks the tokens.
    const int np = PAIRED ? 2 * R.P / VEC : R.P / VEC, nu = np + (R.D - 2 * R.P) / VEC;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const int H = R.heads[w], per = H * nu;
        if (per == 0) continue;
        const T *x = reinterpret_cast<const T *>(R.x[w]);
        T *y = reinterpret_cast<T *>(R.y[w]) + t0 * H * R.D;
        const int rows = per >= NT ? 1 : NT / per;              // tokens side by side
        const int tf = per >= NT ? 0 : (int)threadIdx.x / per, u0 = per >= NT ? (int)threadIdx.x : (int)threadIdx.x - tf * per;
        if (tf >= rows) continue;
        for (int u = u0; u < per; u += NT) {
            const int h = u / nu, k = u - h * nu;
            const T *xh = x + h * R.xh[w];
            for (int t = tf; t < nt; t += rows) {
                const T *src = xh + src_at[w][t];
                T *dst = y + ((int64_t)t * H + h) * R.D;
                float v[VEC];
                if (k >= np) {
                    const int c = 2 * R.P + (k - np) * VEC;
                    load_f32<T, VEC>(src + c, v);
                    store_f32<T, VEC>(dst + c, v);
                } else if (PAIRED) {                            // VEC is even: VEC / 2 neighbouring pairs
                    load_f32<T, VEC>(src + k * VEC, v);
                    const float2 *e = cs + t * R.P + k * (VEC / 2);
#pragma unroll
                    for (int i = 0; i < VEC / 2; ++i) {
                        const float a = v[2 * i], d = v[2 * i + 1];
                        v[2 * i] = fmaf(a, e[i].x, -(d * e[i].y));
                        v[2 * i + 1] = fmaf(d, e[i].x, a * e[i].y);
                    }
                    store_f32<T, VEC>(dst + k * VEC, v);
                } else {
                    float d[VEC];
                    load_f32<T, VEC>(src + k * VEC, v);
                    load_f32<T, VEC>(src + R.P + k * VEC, d);
                    const float2 *e = cs + t * R.P + k * VEC;
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        const float a = v[i], b2 = d[i];
                        v[i] = fmaf(a, e[i].x, -(b2 * e[i].y));
                        d[i] = fmaf(b2, e[i].x, a * e[i].y);
                    }
                    store_f32<T, VEC>(dst + k * VEC, v);
                    store_f32<T, VEC>(dst + R.P + k * VEC, d);
                }
            }
        }
    }
}
}  // namespace

extern "C" int sqd_rotary_axes(const sqd_rotary_args *a) {
    SQD_CHECK_ARG(a, "sqd_rotary_axes: null argument block");
    SQD_CHECK_ARG(a->B >= 0 && a->S >= 0 && a->Hq >= 0 && a->Hk >= 0 && a->D > 0 && a->D <= 1024, "sqd_rotary_axes: bad shape B=%d S=%d Hq=%d Hk=%d D=%d",
                  a->B, a->S, a->Hq, a->Hk, a->D);
    SQD_CHECK_ARG(a->axes >= 1 && a->axes <= MAX_AXES, "sqd_rotary_axes: %d axes (1..%d)", a->axes, MAX_AXES);
    SQD_CHECK_ARG(a->pos_bytes == 4 || a->pos_bytes == 8, "sqd_rotary_axes: positions of %d bytes (4 | 8)", a->pos_bytes);
    RotaryArgs R{};
    int P = 0;
    for (int i = 0; i < a->axes; ++i) {
        SQD_CHECK_ARG(a->pairs[i] >= 0 && a->pairs[i] <= a->D / 2, "sqd_rotary_axes: axis %d has %d pairs", i, a->pairs[i]);
        P += a->pairs[i];
        R.axis_end[i] = P;
    }
    // (a token's pieces are counted in 32 bits, one stride past their number)
    SQD_CHECK_ARG((int64_t)a->Hq * a->D <= (1 << 30) && (int64_t)a->Hk * a->D <= (1 << 30), "sqd_rotary_axes: %d / %d heads of %d features", a->Hq, a->Hk, a->D);
    SQD_CHECK_ARG(P >= 1 && 2 * P <= a->D && a->D % 2 == 0, "sqd_rotary_axes: %d pairs in %d features", P, a->D);
    const int64_t BS = (int64_t)a->B * a->S;
    if (BS == 0 || a->Hq + a->Hk == 0) return SQD_OK;
    SQD_CHECK_ARG(a->pos && a->freq && (a->Hq == 0 || (a->q && a->q_out)) && (a->Hk == 0 || (a->k && a->k_out)), "sqd_rotary_axes: null pointer");
    SQD_CHECK_ARG((a->q != a->q_out || !a->q) && (a->k != a->k_out || !a->k), "sqd_rotary_axes: outputs must not be the inputs");
    R.x[0] = a->q, R.x[1] = a->k, R.y[0] = a->q_out, R.y[1] = a->k_out;
    R.heads[0] = a->Hq, R.heads[1] = a->Hk;
    for (int i = 0; i < 3; ++i) {
        (i == 0 ? R.xb : i == 1 ? R.xs : R.xh)[0] = a->q_stride[i];
        (i == 0 ? R.xb : i == 1 ? R.xs : R.xh)[1] = a->k_stride[i];
    }
    R.pos = a->pos, R.pos_b = a->pos_batch_stride, R.freq = a->freq;
    R.S = a->S, R.D = a->D, R.P = P, R.A = a->axes, R.BS = BS, R.sign = a->inverse ? -1.f : 1.f;
    // tokens per workgroup: 8 (one round of the trigonometry feeds 8 tokens of traffic), 1 while that leaves CUs without work
    R.tokens = BS >= 8 * 512 ? 8 : 1;
    return for_dtype(a->dtype, [&](auto t) {
        using T = decltype(t);
        constexpr int V = 16 / sizeof(T);
        bool vec = a->D % V == 0 && (a->interleaved ? 2 * P % V == 0 : P % V == 0);
        for (int w = 0; w < 2; ++w)
            if (R.heads[w]) vec = vec && aligned16(R.x[w]) && aligned16(R.y[w]) && R.xb[w] % V == 0 && R.xs[w] % V == 0 && R.xh[w] % V == 0;
        for (int w = 0; w < 2; ++w)                              // the interleaved pairs are read as one piece of two elements
            if (R.heads[w] && a->interleaved)
                SQD_CHECK_ARG((uintptr_t)R.x[w] % (2 * sizeof(T)) == 0 && (uintptr_t)R.y[w] % (2 * sizeof(T)) == 0 && R.xb[w] % 2 == 0 &&
                                  R.xs[w] % 2 == 0 && R.xh[w] % 2 == 0, "sqd_rotary_axes: interleaved pairs must not straddle their alignment");
        const size_t lds = (size_t)R.tokens * P * sizeof(float2);
        auto go = [&](auto idx) {
            using I = decltype(idx);
            const dim3 blk(NT);
            const hipStream_t st = (hipStream_t)a->stream;
            for (R.first = 0; R.first < BS; R.first += max_blocks(NT) * R.tokens) {
                const dim3 grid((unsigned)std::min((BS - R.first + R.tokens - 1) / R.tokens, max_blocks(NT)));
                if (a->interleaved) {
                    if (vec) hipLaunchKernelGGL((rotary_kernel<T, I, V, true>), grid, blk, lds, st, R);
                    else hipLaunchKernelGGL((rotary_kernel<T, I, 2, true>), grid, blk, lds, st, R);
                } else {
                    if (vec) hipLaunchKernelGGL((rotary_kernel<T, I, V, false>), grid, blk, lds, st, R);
                    else hipLaunchKernelGGL((rotary_kernel<T, I, 1, false>), grid, blk, lds, st, R);
                }
            }
            SQD_CHECK_LAUNCH("sqd_rotary_axes");
            return SQD_OK;
        };
        return a->pos_bytes == 8 ? go(int64_t{}) : go(int32_t{});
    });
}
