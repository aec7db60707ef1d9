// token_norm.hip — residual addition + root-mean-square norm of token rows [rows, C] and its backward (include/sqd.h section 20).
//
//   stream s = round_T(x + residual)           the sum is kept in the rows' type: it is the residual stream the next layer adds to, and the
//                                              norm and the backward read that same rounded value
//   y_c = w_c s_c r,   r = 1 / sqrt(mean_c s_c^2 + eps)
//   backward, h = g_y w, x^ = s r:   g_x = g_residual = g_s + r (h - x^ mean_c(h x^)),   g_w = sum_rows g_y x^
//
// HBM bound: a row is read once, kept in registers between the sum of squares and the scaling, and written once (forward 4 tensors, backward
// 4).  One wave owns a row of up to 64 x 4 pieces of 16 bytes, so the row sum is one wave reduction and four rows are in flight per workgroup;
// wider rows take the whole workgroup.  Sums in fp32.  g_w: every workgroup of the backward walks rows blockIdx, blockIdx + grid, ... with the
// column sums in registers and leaves one partial row; a second launch adds the partials in a fixed order (no atomics: the same bits every
// run).
// Measured: forward 163840 x 2048 fp16 475 us = 5.6 TB/s (a plain copy of 4 GiB runs at 5.0 TB/s, read + write); 5760 x 768 bf16, in the caches:
// forward 8 us, backward 10 us (3.5 TB/s), sum of the 512 partial rows 3.9 us; 5124 x 1001 fp32, one element a load: 18 / 20 us (4.6 / 4.1 TB/s).
#include "sqd_vec.h"

namespace {
using namespace sqd;

constexpr int NT = 256;

// sum over the LANES threads that share a row; `red` (one slot per wave) is used by whole-workgroup rows only
template <int LANES> __device__ __forceinline__ float row_sum(float v, float *red) {
    v = wave_sum(v);
    if (LANES == 64) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return red[0] + red[1] + red[2] + red[3];
}

template <typename T, typename W, int LANES, int VEC, int NC>
__global__ __launch_bounds__(NT) void norm_fwd_kernel(const T *__restrict__ x, const T *__restrict__ res, const W *__restrict__ w, T *__restrict__ y,
                                                      T *__restrict__ stream, float *__restrict__ rstd, int64_t rows, int C, float eps) {
    __shared__ float red[4];
    const int lane = threadIdx.x % LANES;
    const int64_t row = (int64_t)blockIdx.x * (NT / LANES) + threadIdx.x / LANES;
    if (row >= rows) return;                                   // LANES == 256: uniform over the workgroup
    const int64_t o = row * C;
    float s[NC][VEC];
    float ss = 0.f;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        const int c = (n * LANES + lane) * VEC;
        if (c < C) {
            load_f32<T, VEC>(x + o + c, s[n]);
            if (res) {
                float r[VEC];
                load_f32<T, VEC>(res + o + c, r);
#pragma unroll
                for (int i = 0; i < VEC; ++i) s[n][i] = to_f32(from_f32<T>(s[n][i] + r[i]));
                store_f32<T, VEC>(stream + o + c, s[n]);
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) ss = fmaf(s[n][i], s[n][i], ss);
        }
    }
    const float r = 1.0f / sqrtf(row_sum<LANES>(ss, red) / (float)C + eps);
    if (rstd && lane == 0) rstd[row] = r;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        const int c = (n * LANES + lane) * VEC;
        if (c < C) {
            float wv[VEC];
            load_f32<W, VEC>(w + c, wv);
#pragma unroll
            for (int i = 0; i < VEC; ++i) wv[i] = s[n][i] * r * wv[i];
            store_f32<T, VEC>(y + o + c, wv);
        }
    }
}

// rows of any width: the row is read twice (the second time from the caches)
template <typename T, typename W>
__global__ __launch_bounds__(NT) void norm_fwd_any_kernel(const T *x, const T *res, const W *__restrict__ w, T *y, T *stream, float *__restrict__ rstd,
                                                          int64_t rows, int C, float eps) {
    __shared__ float red[4];
    const int64_t o = (int64_t)blockIdx.x * C;
    float ss = 0.f;
    for (int c = threadIdx.x; c < C; c += NT) {
        float v = to_f32(x[o + c]);
        if (res) {
            const T t = from_f32<T>(v + to_f32(res[o + c]));
            stream[o + c] = t;
            v = to_f32(t);
        }
        ss = fmaf(v, v, ss);
    }
    const float r = 1.0f / sqrtf(row_sum<NT>(ss, red) / (float)C + eps);
    if (rstd && threadIdx.x == 0) rstd[blockIdx.x] = r;
    for (int c = threadIdx.x; c < C; c += NT) {
        float v = to_f32(x[o + c]);
        if (res) v = to_f32(from_f32<T>(v + to_f32(res[o + c])));
        y[o + c] = from_f32<T>(v * r * to_f32(w[c]));
    }
}

template <typename T, typename W, int LANES, int VEC, int NC>
__global__ __launch_bounds__(NT) void norm_bwd_kernel(const T *__restrict__ gy, const T *__restrict__ gs, const T *__restrict__ s_, const W *__restrict__ w,
                                                      const float *__restrict__ rstd, T *__restrict__ gx, float *__restrict__ part, int64_t rows, int C) {
    constexpr int RP = NT / LANES;
    __shared__ float red[RP == 1 ? 4 : (RP - 1) * NC * VEC * 64];
    const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    float wv[NC][VEC], dw[NC][VEC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        const int c = (n * LANES + lane) * VEC;
#pragma unroll
        for (int i = 0; i < VEC; ++i) dw[n][i] = wv[n][i] = 0.f;
        if (c < C) load_f32<W, VEC>(w + c, wv[n]);
    }
    for (int64_t row = (int64_t)blockIdx.x * RP + sub; row < rows; row += (int64_t)gridDim.x * RP) {
        const int64_t o = row * C;
        const float r = rstd[row];
        float xh[NC][VEC], h[NC][VEC], g[NC][VEC];
        float dot = 0.f;
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            const int c = (n * LANES + lane) * VEC;
            if (c < C) {
                load_f32<T, VEC>(s_ + o + c, xh[n]);
                load_f32<T, VEC>(gy + o + c, h[n]);
                if (gs) load_f32<T, VEC>(gs + o + c, g[n]);
            }
        }
#pragma unroll
        for (int n = 0; n < NC; ++n)
            if ((n * LANES + lane) * VEC < C) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    xh[n][i] *= r;
                    dw[n][i] = fmaf(h[n][i], xh[n][i], dw[n][i]);
                    h[n][i] *= wv[n][i];
                    dot = fmaf(h[n][i], xh[n][i], dot);
                }
            }
        const float m = row_sum<LANES>(dot, red) / (float)C;
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            const int c = (n * LANES + lane) * VEC;
            if (c < C) {
                float out[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) out[i] = fmaf(r, h[n][i] - xh[n][i] * m, gs ? g[n][i] : 0.f);
                store_f32<T, VEC>(gx + o + c, out);
            }
        }
    }
    if (RP > 1) {                                               // the waves' column sums, added in wave order
        if (sub > 0)
#pragma unroll
            for (int n = 0; n < NC; ++n)
#pragma unroll
                for (int i = 0; i < VEC; ++i) red[((sub - 1) * NC * VEC + n * VEC + i) * 64 + lane] = dw[n][i];
        __syncthreads();
        if (sub > 0) return;
#pragma unroll
        for (int n = 0; n < NC; ++n)
#pragma unroll
            for (int i = 0; i < VEC; ++i)
#pragma unroll
                for (int k = 0; k < RP - 1; ++k) dw[n][i] += red[(k * NC * VEC + n * VEC + i) * 64 + lane];
    }
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        const int c = (n * LANES + lane) * VEC;
        if (c < C)
#pragma unroll
            for (int i = 0; i < VEC; ++i) part[(int64_t)blockIdx.x * C + c + i] = dw[n][i];
    }
}

// rows of any width: g_x row by row, reading the row twice ...
template <typename T, typename W>
__global__ __launch_bounds__(NT) void norm_bwd_any_kernel(const T *__restrict__ gy, const T *__restrict__ gs, const T *__restrict__ s_, const W *__restrict__ w,
                                                          const float *__restrict__ rstd, T *__restrict__ gx, int C) {
    __shared__ float red[4];
    const int64_t o = (int64_t)blockIdx.x * C;
    const float r = rstd[blockIdx.x];
    float dot = 0.f;
    for (int c = threadIdx.x; c < C; c += NT) dot = fmaf(to_f32(gy[o + c]) * to_f32(w[c]), to_f32(s_[o + c]) * r, dot);
    const float m = row_sum<NT>(dot, red) / (float)C;
    for (int c = threadIdx.x; c < C; c += NT) {
        const float h = to_f32(gy[o + c]) * to_f32(w[c]), xh = to_f32(s_[o + c]) * r;
        gx[o + c] = from_f32<T>(fmaf(r, h - xh * m, gs ? to_f32(gs[o + c]) : 0.f));
    }
}
// ... and the column sums of g_y x^ in a launch of their own: block = 64 columns x 4 row groups, blockIdx.y = one partial row
template <typename T>
__global__ __launch_bounds__(NT) void norm_gw_any_kernel(const T *__restrict__ gy, const T *__restrict__ s_, const float *__restrict__ rstd,
                                                         float *__restrict__ part, int64_t rows, int C) {
    __shared__ float red[4][64];
    const int col = threadIdx.x & 63, grp = threadIdx.x >> 6, c = blockIdx.x * 64 + col;
    float a = 0.f;
    if (c < C)
        for (int64_t row = (int64_t)blockIdx.y * 4 + grp; row < rows; row += (int64_t)gridDim.y * 4)
            a = fmaf(to_f32(gy[row * C + c]), to_f32(s_[row * C + c]) * rstd[row], a);
    red[grp][col] = a;
    __syncthreads();
    if (grp == 0 && c < C) part[(int64_t)blockIdx.y * C + c] = red[0][col] + red[1][col] + red[2][col] + red[3][col];
}

// g_w[c] = sum of the partial rows, in a fixed order: 16 columns x 16 row groups, eight loads of a group under way at a time, then a tree over the
// groups
template <typename W>
__global__ __launch_bounds__(NT) void norm_gw_reduce_kernel(const float *__restrict__ part, W *__restrict__ gw, int nparts, int C) {
    __shared__ float red[16][17];
    const int col = threadIdx.x & 15, grp = threadIdx.x >> 4, c = blockIdx.x * 16 + col;
    float a[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (c < C) {
        int p = grp;
        for (; p + 16 * 7 < nparts; p += 16 * 8)
#pragma unroll
            for (int k = 0; k < 8; ++k) a[k] += part[(int64_t)(p + 16 * k) * C + c];
        for (; p < nparts; p += 16) a[0] += part[(int64_t)p * C + c];
    }
    red[grp][col] = ((a[0] + a[1]) + (a[2] + a[3])) + ((a[4] + a[5]) + (a[6] + a[7]));
    __syncthreads();
#pragma unroll
    for (int k = 8; k > 0; k >>= 1) {
        if (grp < k) red[grp][col] += red[grp + k][col];
        __syncthreads();
    }
    if (grp == 0 && c < C) gw[c] = from_f32<W>(red[0][col]);
}

// the row layout for a width: f(lanes, vec, nc) as compile-time constants; lanes 0 = the any-width kernels
template <int L, int V, int N> struct RowLayout { static constexpr int lanes = L, vec = V, nc = N; };
template <typename T, typename F> int for_layout(int C, bool vec_ok, F &&f) {
    constexpr int V = 16 / sizeof(T);
    if (vec_ok) {
        if (C <= 64 * V) return f(RowLayout<64, V, 1>{});
        if (C <= 128 * V) return f(RowLayout<64, V, 2>{});
        if (C <= 256 * V) return f(RowLayout<64, V, 4>{});
        if (C <= 512 * V) return f(RowLayout<256, V, 2>{});
        if (C <= 1024 * V) return f(RowLayout<256, V, 4>{});
    } else {
        if (C <= 256) return f(RowLayout<64, 1, 4>{});
        if (C <= 1024) return f(RowLayout<64, 1, 16>{});
        if (C <= 4096) return f(RowLayout<256, 1, 16>{});
    }
    return f(RowLayout<0, 1, 1>{});
}

int check_norm(const char *who, int64_t rows, int C, int dtype, int wdtype) {
    // (C: column counters run one stride past it, and the weight gradient takes 16 threads a column)
    SQD_CHECK_ARG(rows >= 0 && rows <= (1ll << 30) && C > 0 && C <= (1 << 27), "%s: bad shape rows=%lld C=%d", who, (long long)rows, C);
    SQD_CHECK_ARG(dtype >= SQD_F32 && dtype <= SQD_F16 && (wdtype == dtype || wdtype == SQD_F32), "%s: element types %d / weight %d unsupported", who, dtype,
                  wdtype);
    return SQD_OK;
}
}  // namespace

extern "C" int sqd_rms_norm_fwd(const void *x, const void *res, const void *w, void *y, void *stream_out, float *rstd, int64_t rows, int C, float eps,
                                int dtype, int wdtype, void *stream) {
    if (int e = check_norm("sqd_rms_norm_fwd", rows, C, dtype, wdtype)) return e;
    if (rows == 0) return SQD_OK;
    SQD_CHECK_ARG(x && w && y && (!res == !stream_out), "sqd_rms_norm_fwd: null pointer (a residual comes with a stream output)");
    SQD_CHECK_ARG(eps >= 0.f, "sqd_rms_norm_fwd: eps=%g", (double)eps);
    return for_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto wt) {
            using W = decltype(wt);
            const bool vec = C % (16 / sizeof(T)) == 0 && aligned16(x) && aligned16(res) && aligned16(w) && aligned16(y) && aligned16(stream_out);
            return for_layout<T>(C, vec, [&](auto lay) {
                using L = decltype(lay);
                constexpr int RP = L::lanes ? NT / (L::lanes ? L::lanes : 1) : 1;              // rows of a workgroup
                for (int64_t r0 = 0; r0 < rows; r0 += max_blocks(NT) * RP) {
                    const int64_t n = std::min(rows - r0, max_blocks(NT) * RP), o = r0 * C;
                    const dim3 grid((unsigned)((n + RP - 1) / RP));
                    const T *xr = (const T *)x + o, *rr = res ? (const T *)res + o : nullptr;
                    T *yr = (T *)y + o, *sr = stream_out ? (T *)stream_out + o : nullptr;
                    float *rs = rstd ? rstd + r0 : nullptr;
                    if constexpr (L::lanes == 0)
                        hipLaunchKernelGGL((norm_fwd_any_kernel<T, W>), grid, dim3(NT), 0, (hipStream_t)stream, xr, rr, (const W *)w, yr, sr, rs, n, C, eps);
                    else
                        hipLaunchKernelGGL((norm_fwd_kernel<T, W, L::lanes, L::vec, L::nc>), grid, dim3(NT), 0, (hipStream_t)stream, xr, rr, (const W *)w, yr,
                                           sr, rs, n, C, eps);
                }
                SQD_CHECK_LAUNCH("sqd_rms_norm_fwd");
                return SQD_OK;
            });
        };
        return wdtype == SQD_F32 ? go(float{}) : go(t);
    });
}

// partial rows of g_w: enough workgroups to fill 256 CUs twice, fewer when there are fewer rows to walk
extern "C" int sqd_rms_norm_nblk(int64_t rows) { return rows < 1 ? 1 : (int)(rows < 2048 ? (rows + 3) / 4 : 512); }

extern "C" int sqd_rms_norm_bwd(const void *gy, const void *gs, const void *s, const void *w, const float *rstd, void *gx, void *gw, float *part,
                                int64_t rows, int C, int dtype, int wdtype, void *stream) {
    if (int e = check_norm("sqd_rms_norm_bwd", rows, C, dtype, wdtype)) return e;
    SQD_CHECK_ARG(gw && part && w && (rows == 0 || (gy && s && rstd && gx)), "sqd_rms_norm_bwd: null pointer");
    const int nblk = sqd_rms_norm_nblk(rows);
    const hipStream_t st = (hipStream_t)stream;
    return for_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto wt) {
            using W = decltype(wt);
            const bool vec = C % (16 / sizeof(T)) == 0 && aligned16(gy) && aligned16(gs) && aligned16(s) && aligned16(w) && aligned16(gx);
            const int rc = for_layout<T>(C, vec, [&](auto lay) {
                using L = decltype(lay);
                if constexpr (L::lanes == 0) {
                    SQD_CHECK_ARG(rows <= max_blocks(NT), "sqd_rms_norm_bwd: %lld rows of %d features", (long long)rows, C);
                    if (rows)
                        hipLaunchKernelGGL((norm_bwd_any_kernel<T, W>), dim3((unsigned)rows), dim3(NT), 0, st, (const T *)gy, (const T *)gs, (const T *)s,
                                           (const W *)w, rstd, (T *)gx, C);
                    SQD_CHECK_LAUNCH("sqd_rms_norm_bwd");
                    hipLaunchKernelGGL((norm_gw_any_kernel<T>), dim3((C + 63) / 64, nblk), dim3(NT), 0, st, (const T *)gy, (const T *)s, rstd, part, rows, C);
                } else {
                    hipLaunchKernelGGL((norm_bwd_kernel<T, W, L::lanes, L::vec, L::nc>), dim3(nblk), dim3(NT), 0, st, (const T *)gy, (const T *)gs,
                                       (const T *)s, (const W *)w, rstd, (T *)gx, part, rows, C);
                }
                SQD_CHECK_LAUNCH("sqd_rms_norm_bwd");
                return SQD_OK;
            });
            if (rc) return rc;
            hipLaunchKernelGGL((norm_gw_reduce_kernel<W>), dim3((C + 15) / 16), dim3(NT), 0, st, part, (W *)gw, nblk, C);
            SQD_CHECK_LAUNCH("sqd_rms_norm_bwd");
            return SQD_OK;
        };
        return wdtype == SQD_F32 ? go(float{}) : go(t);
    });
}
