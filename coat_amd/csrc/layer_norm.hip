// LayerNorm over the last dimension of bf16 / fp16 / fp32 tensors, forward and backward, beside the FP8 LayerNorm of
// layernorm.hip (whose input is per-group FP8 and whose output feeds a per-tensor quantizer).
//
//   forward    mean = sum(x) / N;  rstd = 1 / sqrt(sum((x - mean)^2) / N + eps);  y = (x - mean) * rstd (* w (+ b))
//   backward   h = (x - mean) * rstd;  t = dy * w;  dx = rstd * (t - mean(t) - h * mean(t * h))
//              dw = sum over rows of dy * h;  db = sum over rows of dy
// All sums are fp32; the variance is the two-pass one (no cancellation for rows far from zero).  Outputs are rounded once, to
// x's type (y, dx) and the weight's (dw, db).  dw / db: every block sums its own rows into one fp32 partial row, a second
// kernel adds the partial rows in a fixed order: no atomics, the same bits on every run.
#include <math.h>

#include "coat_host.h"
#include "elem_io.h"

namespace coat {

// Sum over a block of W waves, in every thread; `red` holds W floats and may be reused after the next barrier of the caller.
template <int W> __device__ __forceinline__ float block_sum(float v, float* red) {
    v = cluster_sum<64>(v);
    if (W == 1) return v;
    __syncthreads();  // an earlier reduction may still be reading
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = red[0];
#pragma unroll
    for (int k = 1; k < W; k++) s += red[k];
    return s;
}

// ------------------------------------------------------------------------------------------------ rows of any length
// One block per row, the row read once per pass (the second and third reads hit the L2).
template <int DT>
__global__ __launch_bounds__(256) void k_ln_fwd_long(const void* __restrict__ x, int64_t x_pitch, const void* __restrict__ w,
                                                     const void* __restrict__ b, int w_dt, void* __restrict__ y,
                                                     float* __restrict__ mean_out, float* __restrict__ rstd_out, int64_t M, int64_t N,
                                                     float eps) {
    __shared__ float red[4];
    for (int64_t row = blockIdx.x; row < M; row += gridDim.x) {
        const void* xr = elem_at<DT>(x, row * x_pitch);
        float v[8], s = 0.0f;
        for (int64_t c = threadIdx.x * 8; c < N; c += 256 * 8) {
            load8<DT>(elem_at<DT>(xr, c), N - c, v);
#pragma unroll
            for (int i = 0; i < 8; i++) s += v[i];
        }
        const float mean = block_sum<4>(s, red) / (float)N;
        s = 0.0f;
        for (int64_t c = threadIdx.x * 8; c < N; c += 256 * 8) {
            load8<DT>(elem_at<DT>(xr, c), N - c, v);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float d = c + i < N ? v[i] - mean : 0.0f;
                s = fmaf(d, d, s);
            }
        }
        const float rstd = 1.0f / sqrtf(block_sum<4>(s, red) / (float)N + eps);
        void* yr = elem_at<DT>(y, row * N);
        for (int64_t c = threadIdx.x * 8; c < N; c += 256 * 8) {
            float wv[8], bv[8];
            load8<DT>(elem_at<DT>(xr, c), N - c, v);
            if (w) load8_rt(w, w_dt, c, N, wv);
            if (b) load8_rt(b, w_dt, c, N, bv);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                v[i] = (v[i] - mean) * rstd;
                if (w) v[i] *= wv[i];
                if (b) v[i] += bv[i];
            }
            store8<DT>(elem_at<DT>(yr, c), N - c, v);
        }
        if (threadIdx.x == 0) {
            mean_out[row] = mean;
            rstd_out[row] = rstd;
        }
    }
}

template <int DT>
__global__ __launch_bounds__(256) void k_ln_bwd_long(const void* __restrict__ dy, int64_t dy_pitch, const void* __restrict__ x,
                                                     int64_t x_pitch, const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                                                     const void* __restrict__ w, int w_dt, void* __restrict__ dx, int64_t M, int64_t N) {
    __shared__ float red[4];
    for (int64_t row = blockIdx.x; row < M; row += gridDim.x) {
        const void *xr = elem_at<DT>(x, row * x_pitch), *gr = elem_at<DT>(dy, row * dy_pitch);
        void* dr = elem_at<DT>(dx, row * N);
        const float mean = mean_in[row], rstd = rstd_in[row];
        float v[8], t[8], wv[8], st = 0.0f, sth = 0.0f;
        for (int64_t c = threadIdx.x * 8; c < N; c += 256 * 8) {
            load8<DT>(elem_at<DT>(xr, c), N - c, v);
            load8<DT>(elem_at<DT>(gr, c), N - c, t);  // zeros past the end: they add nothing to either sum
            if (w) load8_rt(w, w_dt, c, N, wv);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if (w) t[i] *= wv[i];
                st += t[i];
                sth = fmaf(t[i], (v[i] - mean) * rstd, sth);
            }
        }
        const float mt = block_sum<4>(st, red) / (float)N, mth = block_sum<4>(sth, red) / (float)N;
        for (int64_t c = threadIdx.x * 8; c < N; c += 256 * 8) {
            load8<DT>(elem_at<DT>(xr, c), N - c, v);
            load8<DT>(elem_at<DT>(gr, c), N - c, t);
            if (w) load8_rt(w, w_dt, c, N, wv);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if (w) t[i] *= wv[i];
                v[i] = (t[i] - mt - (v[i] - mean) * rstd * mth) * rstd;
            }
            store8<DT>(elem_at<DT>(dr, c), N - c, v);
        }
    }
}

// Partial rows of dw and db: block (i, j) sums the rows j, j + gridDim.y, ... of the 2048 columns from 2048 i.
template <int DT>
__global__ __launch_bounds__(256) void k_ln_bwd_wb_long(const void* __restrict__ dy, int64_t dy_pitch, const void* __restrict__ x,
                                                        int64_t x_pitch, const float* __restrict__ mean_in,
                                                        const float* __restrict__ rstd_in, float* __restrict__ pw, float* __restrict__ pb,
                                                        int64_t M, int64_t N) {
    const int64_t c = (int64_t)blockIdx.x * 2048 + threadIdx.x * 8;
    if (c >= N) return;
    float aw[8], ab[8];
#pragma unroll
    for (int i = 0; i < 8; i++) aw[i] = ab[i] = 0.0f;
    for (int64_t row = blockIdx.y; row < M; row += gridDim.y) {
        float v[8], g[8];
        load8<DT>(elem_at<DT>(x, row * x_pitch + c), N - c, v);
        load8<DT>(elem_at<DT>(dy, row * dy_pitch + c), N - c, g);
        const float mean = mean_in[row], rstd = rstd_in[row];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            aw[i] = fmaf(g[i], (v[i] - mean) * rstd, aw[i]);
            ab[i] += g[i];
        }
    }
    if (pw) store8<kF32>(pw + blockIdx.y * N + c, N - c, aw);
    if (pb) store8<kF32>(pb + blockIdx.y * N + c, N - c, ab);
}

// ------------------------------------------------------------------------------------------------ dw, db from partial rows
// 32 columns a block (one 128-byte line of each partial row); 16 slices of threads take the rows in turn, slice sums are
// added in slice order.  blockIdx.y: 0 = the first pair given, 1 = the second.
constexpr int kSumCols = 32, kSumSlices = 16;
__global__ __launch_bounds__(kSumCols* kSumSlices) void k_ln_sum_partials(const float* __restrict__ pw, void* __restrict__ dw,
                                                                         const float* __restrict__ pb, void* __restrict__ db, int dt,
                                                                         int64_t rows, int64_t N) {
    __shared__ float red[kSumSlices][kSumCols];
    const int col = threadIdx.x % kSumCols, slice = threadIdx.x / kSumCols;
    const int64_t c = (int64_t)blockIdx.x * kSumCols + col;
    const float* p = blockIdx.y == 0 && dw ? pw : pb;
    void* out = blockIdx.y == 0 && dw ? dw : db;
    float s = 0.0f;
    if (c < N)
        for (int64_t r = slice; r < rows; r += kSumSlices) s += p[r * N + c];
    red[slice][col] = s;
    __syncthreads();
    if (slice == 0 && c < N) {
        s = red[0][col];
#pragma unroll
        for (int k = 1; k < kSumSlices; k++) s += red[k][col];
        if (dt == kF32) store_from_f32<kF32>(out, c, s);
        else if (dt == kBF16) store_from_f32<kBF16>(out, c, s);
        else store_from_f32<kF16>(out, c, s);
    }
}

}  // namespace coat

using namespace coat;

static bool ln_dtype(int dt) { return dt == COAT_F32 || dt == COAT_BF16 || dt == COAT_F16; }
static bool ln_aligned(const void* p, int dt) { return ((uintptr_t)p & (dt == COAT_F32 ? 3u : 1u)) == 0; }

extern "C" int coat_layer_norm_forward(const void* x, int64_t x_pitch, int x_dtype, const void* w, const void* b, int w_dtype,
                                       void* y, float* mean, float* rstd, int64_t M, int64_t N, float eps, void* stream) {
    if (!ln_dtype(x_dtype) || (w && !ln_dtype(w_dtype))) return COAT_EDTYPE;
    if (M < 0 || N <= 0 || !(eps >= 0.0f) || (b && !w)) return COAT_EINVAL;
    if (x_pitch == 0) x_pitch = N;
    if (x_pitch < N) return COAT_ESHAPE;
    if (M == 0) return COAT_OK;
    if (!x || !y || !mean || !rstd) return COAT_EINVAL;
    if (!ln_aligned(x, x_dtype) || !ln_aligned(y, x_dtype) || !ln_aligned(mean, COAT_F32) || !ln_aligned(rstd, COAT_F32) ||
        (w && !ln_aligned(w, w_dtype)) || (b && !ln_aligned(b, w_dtype)))
        return COAT_EALIGN;
    const dim3 grid((unsigned)(M < 65536 ? M : 65536));
    hipStream_t st = (hipStream_t)stream;
    if (x_dtype == COAT_F32)
        hipLaunchKernelGGL((k_ln_fwd_long<kF32>), grid, dim3(256), 0, st, x, x_pitch, w, b, w_dtype, y, mean, rstd, M, N, eps);
    else if (x_dtype == COAT_BF16)
        hipLaunchKernelGGL((k_ln_fwd_long<kBF16>), grid, dim3(256), 0, st, x, x_pitch, w, b, w_dtype, y, mean, rstd, M, N, eps);
    else
        hipLaunchKernelGGL((k_ln_fwd_long<kF16>), grid, dim3(256), 0, st, x, x_pitch, w, b, w_dtype, y, mean, rstd, M, N, eps);
    return coat_launch_status();
}

extern "C" int coat_layer_norm_partials(int64_t M, int64_t N) {
    if (M < 0 || N <= 0) return COAT_EINVAL;
    return (int)(M < 256 ? (M > 0 ? M : 1) : 256);
}

template <int DT>
static int ln_backward(const void* dy, int64_t dy_pitch, const void* x, int64_t x_pitch, const float* mean, const float* rstd,
                       const void* w, int w_dtype, void* dx, void* dw, void* db, int wb_dtype, float* pw, float* pb, int n_partial,
                       int64_t M, int64_t N, hipStream_t st) {
    if (M > 0) {
        if (dx) {
            hipLaunchKernelGGL((k_ln_bwd_long<DT>), dim3((unsigned)(M < 65536 ? M : 65536)), dim3(256), 0, st, dy, dy_pitch, x, x_pitch, mean,
                               rstd, w, w_dtype, dx, M, N);
            if (const int rc = coat_launch_status()) return rc;
        }
        if (dw || db) {
            hipLaunchKernelGGL((k_ln_bwd_wb_long<DT>), dim3((unsigned)((N + 2047) / 2048), (unsigned)n_partial), dim3(256), 0, st, dy, dy_pitch, x,
                               x_pitch, mean, rstd, dw ? pw : nullptr, db ? pb : nullptr, M, N);
            if (const int rc = coat_launch_status()) return rc;
        }
    }
    if (dw || db) {
        const int64_t rows = M > 0 ? n_partial : 0;  // no rows: the sums are zeros
        hipLaunchKernelGGL(k_ln_sum_partials, dim3((unsigned)((N + kSumCols - 1) / kSumCols), dw && db ? 2 : 1), dim3(kSumCols * kSumSlices), 0,
                           st, pw, dw, pb, db, wb_dtype, rows, N);
        return coat_launch_status();
    }
    return COAT_OK;
}

extern "C" int coat_layer_norm_backward(const void* dy, int64_t dy_pitch, const void* x, int64_t x_pitch, int x_dtype, const float* mean,
                                        const float* rstd, const void* w, int w_dtype, void* dx, void* dw, void* db, float* partial,
                                        int n_partial, int64_t M, int64_t N, void* stream) {
    if (!ln_dtype(x_dtype) || ((w || dw || db) && !ln_dtype(w_dtype))) return COAT_EDTYPE;
    if (M < 0 || N <= 0 || (dw && !w)) return COAT_EINVAL;
    if (N > ((int64_t)1 << 31)) return COAT_ESHAPE;
    if (x_pitch == 0) x_pitch = N;
    if (dy_pitch == 0) dy_pitch = N;
    if (x_pitch < N || dy_pitch < N) return COAT_ESHAPE;
    if ((dw || db) && M > 0 && (!partial || n_partial < 1 || n_partial > 65535)) return COAT_EINVAL;
    if (M > 0 && (!dy || !x || !mean || !rstd)) return COAT_EINVAL;
    if (!ln_aligned(dy, x_dtype) || !ln_aligned(x, x_dtype) || !ln_aligned(dx, x_dtype) || !ln_aligned(mean, COAT_F32) ||
        !ln_aligned(rstd, COAT_F32) || !ln_aligned(partial, COAT_F32) || (w && !ln_aligned(w, w_dtype)) || (dw && !ln_aligned(dw, w_dtype)) ||
        (db && !ln_aligned(db, w_dtype)))
        return COAT_EALIGN;
    if (!dx && !dw && !db) return COAT_OK;
    float* pw = partial;
    float* pb = dw && db ? partial + (int64_t)n_partial * N : partial;
    hipStream_t st = (hipStream_t)stream;
    switch (x_dtype) {
        case COAT_F32:
            return ln_backward<kF32>(dy, dy_pitch, x, x_pitch, mean, rstd, w, w_dtype, dx, dw, db, w_dtype, pw, pb, n_partial, M, N, st);
        case COAT_BF16:
            return ln_backward<kBF16>(dy, dy_pitch, x, x_pitch, mean, rstd, w, w_dtype, dx, dw, db, w_dtype, pw, pb, n_partial, M, N, st);
        default:
            return ln_backward<kF16>(dy, dy_pitch, x, x_pitch, mean, rstd, w, w_dtype, dx, dw, db, w_dtype, pw, pb, n_partial, M, N, st);
    }
}
