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

#include <type_traits>

#include "coat_host.h"
#include "elem_io.h"
#include "tensor_list.h"

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

// ------------------------------------------------------------------------------------------------ rows held in registers
// L lanes work on a row and hold C pieces of 8 elements each: piece k of lane l begins at column (k lanes + l) 8, so that the
// lanes of a wave read one run of memory.  L = 8 .. 64: a wave works on 64 / L rows at a time and no barrier is needed.
// L = kBlock: the block works on one row with as many waves as that takes.  The weights stay in registers over the rows of a
// block, and the next row's loads are issued before the sums of the present one are exchanged.
// RAGGED: N is not a multiple of 8; the last piece of a row then shares elements with the one before, which its sums leave out.
constexpr int kBlock = 0;
constexpr int form_threads(int L, int C) { return L != kBlock ? 256 : C <= 2 ? 1024 : 512; }  // launch bound
constexpr int form_rows(int L) { return L != kBlock ? 256 / L : 1; }                          // rows at a time

// Sum over the lanes of a row, in each of them.  Block form: `red` holds 16 floats, zero beyond the block's waves; a buffer may be
// used again after another buffer's exchange (whose barrier every wave reaches only after it has read this one).
template <int L> __device__ __forceinline__ float row_sum(float v, float* red) {
    if (L != kBlock) return cluster_sum<L ? L : 1>(v);
    v = cluster_sum<64>(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return cluster_sum<16>(red[threadIdx.x & 15]);
}
// Wave sums of four values, each with the additions of cluster_sum<64>, in three exchanges between 16-lane rows instead of eight:
// row 0 returns the sum of a0, row 1 of a1, row 2 of b0, row 3 of b1.
__device__ __forceinline__ float four_wave_sums(float a0, float a1, float b0, float b1) {
    const bool odd = threadIdx.x & 16, upper = threadIdx.x & 32;
    a0 = cluster_sum<16>(a0);
    a1 = cluster_sum<16>(a1);
    b0 = cluster_sum<16>(b0);
    b1 = cluster_sum<16>(b1);
    const float a = (odd ? a1 : a0) + lane_xor_f32(odd ? a0 : a1, 16), b = (odd ? b1 : b0) + lane_xor_f32(odd ? b0 : b1, 16);
    return (upper ? b : a) + lane_xor_f32(upper ? a : b, 32);
}
template <int DT, int L, int C, bool RAGGED>
__global__ __launch_bounds__(form_threads(L, C)) void k_ln_fwd(const void* __restrict__ x, int64_t x_pitch, const void* __restrict__ w,
                                                                 const void* __restrict__ b, int w_dt, void* __restrict__ y,
                                                                 float* __restrict__ mean_out, float* __restrict__ rstd_out, int64_t M,
                                                                 int N, float eps) {
    constexpr int R = form_rows(L);
    __shared__ float red[2][16];
    const int lanes = L == kBlock ? blockDim.x : L;
    const int l = L == kBlock ? threadIdx.x : threadIdx.x % (L ? L : 1), r = L == kBlock ? 0 : threadIdx.x / (L ? L : 1);
    const int64_t step = (int64_t)gridDim.x * R;
    int64_t row = (int64_t)blockIdx.x * R + r;
    const int64_t rounds = (M - (int64_t)blockIdx.x * R + step - 1) / step;  // the same for the whole block
    const float inv_n = 1.0f / (float)N;
    if (L == kBlock) {
        if (threadIdx.x < 32) red[threadIdx.x >> 4][threadIdx.x & 15] = 0.0f;
        __syncthreads();
    }
    Raw8<DT> raw[C];
    float wv[C][8], bv[C][8];
#pragma unroll
    for (int k = 0; k < C; k++) raw[k] = load_piece<DT, RAGGED, false>(elem_at<DT>(x, row * x_pitch), (k * lanes + l) * 8, N, row < M);
#pragma unroll
    for (int k = 0; k < C; k++) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            wv[k][j] = 1.0f;
            bv[k][j] = 0.0f;
        }
        const int c = (k * lanes + l) * 8, at = RAGGED ? piece_begin(c, N) : c;
        if (w && c < N) load8_rt(w, w_dt, at, N, wv[k]);
        if (b && c < N) load8_rt(b, w_dt, at, N, bv[k]);
    }
    for (int64_t i = 0; i < rounds; i++, row += step) {
        float v[C][8], s = 0.0f;
#pragma unroll
        for (int k = 0; k < C; k++) {
            raw8_to_f32<DT>(raw[k], v[k]);
            float own[8];
#pragma unroll
            for (int j = 0; j < 8; j++) own[j] = !RAGGED || own_element((k * lanes + l) * 8, N, j) ? v[k][j] : 0.0f;
            s += ((own[0] + own[1]) + (own[2] + own[3])) + ((own[4] + own[5]) + (own[6] + own[7]));
        }
        if (i + 1 < rounds) {
            const int64_t next = row + step;
#pragma unroll
            for (int k = 0; k < C; k++)
                raw[k] = load_piece<DT, RAGGED, false>(elem_at<DT>(x, next * x_pitch), (k * lanes + l) * 8, N, next < M);
        }
        const float mean = row_sum<L>(s, red[0]) * inv_n;
        s = 0.0f;
#pragma unroll
        for (int k = 0; k < C; k++) {
            const int c = (k * lanes + l) * 8;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                v[k][j] -= mean;
                const float d = c < N && (!RAGGED || own_element(c, N, j)) ? v[k][j] : 0.0f;
                s = fmaf(d, d, s);
            }
        }
        const float rstd = 1.0f / sqrtf(row_sum<L>(s, red[1]) * inv_n + eps);
        if (row < M) {
#pragma unroll
            for (int k = 0; k < C; k++) {
                const int c = (k * lanes + l) * 8;
                if (c >= N) continue;
#pragma unroll
                for (int j = 0; j < 8; j++) v[k][j] = fmaf(v[k][j] * rstd, wv[k][j], bv[k][j]);
                store8<DT>(elem_at<DT>(y, row * N + (RAGGED ? piece_begin(c, N) : c)), RAGGED ? N : 8, v[k]);
            }
            if (l == 0) {
                mean_out[row] = mean;
                rstd_out[row] = rstd;
            }
        }
    }
}

// x and dy are not needed again after this kernel: streaming loads.  In a training step dy has just been written and x, of the forward,
// has left the caches: [262144, 128] bf16 40 us against 45 with ordinary loads, [8192, 4096] bf16 43 against 50, [8192, 1024] fp32 29
// against 30; with neither in the caches 45 against 70.  Ordinary loads are better off only where both were just written and fit
// (fp32 [8192, 1024] 25 against 28; bf16 as above 40 against 40), which a forward in between rules out.  Streaming x alone: 39, 46, 29.  In the
// forward, whose x the backward reads, streaming costs 24 -> 26.
// dx, and with SUMS the sums for dw and db (either may be NULL): one partial row per block, in pw / pb, or, if there is one block
// only, dw and db themselves.
template <int DT, int L, int C, bool RAGGED, bool SUMS>
__global__ __launch_bounds__(form_threads(L, C)) void k_ln_bwd(const void* __restrict__ dy, int64_t dy_pitch, const void* __restrict__ x,
                                                                 int64_t x_pitch, const float* __restrict__ mean_in,
                                                                 const float* __restrict__ rstd_in, const void* __restrict__ w, int w_dt,
                                                                 void* __restrict__ dx, void* __restrict__ dw, void* __restrict__ db,
                                                                 float* __restrict__ pw, float* __restrict__ pb, int64_t M, int N) {
    constexpr int R = form_rows(L);
    constexpr bool kShared = SUMS && R > 1;  // several rows of the block share a column: summed through LDS at the end
    // Rows of four pieces a lane keep two sums of two pieces each, in the places of the waves that hold those pieces where dx alone is
    // wanted (two pieces a lane, twice the waves): dx has the same bits with and without the parameters' gradients.
    constexpr int H = L == kBlock && C == 4 ? 2 : 1;
    constexpr bool kLean = C * (DT == kF32 ? 2 : 1) * (RAGGED ? 2 : 1) >= 8;  // no registers left for the next row
    __shared__ float red[4][16];
    __shared__ float cols[kShared ? R : 1][kShared ? L * C * 8 : 1];
    const int lanes = L == kBlock ? blockDim.x : L;
    const int l = L == kBlock ? threadIdx.x : threadIdx.x % (L ? L : 1), r = L == kBlock ? 0 : threadIdx.x / (L ? L : 1);
    const int64_t step = (int64_t)gridDim.x * R;
    int64_t row = (int64_t)blockIdx.x * R + r;
    const int64_t rounds = (M - (int64_t)blockIdx.x * R + step - 1) / step;
    const float inv_n = 1.0f / (float)N;
    if (L == kBlock) {
        if (threadIdx.x < 64) red[threadIdx.x >> 4][threadIdx.x & 15] = 0.0f;
        __syncthreads();
    }
    float wv[C][8], aw[C][8], ab[C][8];
    Raw8<DT> rx[C], rg[C];
    float mean, rstd;
    auto load = [&](int64_t at) {
#pragma unroll
        for (int k = 0; k < C; k++) {
            const int c = (k * lanes + l) * 8;
            rx[k] = load_piece<DT, RAGGED, true>(elem_at<DT>(x, at * x_pitch), c, N, at < M);
            rg[k] = load_piece<DT, RAGGED, true>(elem_at<DT>(dy, at * dy_pitch), c, N, at < M);
        }
        mean = at < M ? mean_in[at] : 0.0f;
        rstd = at < M ? rstd_in[at] : 0.0f;
    };
    if (!kLean) load(row);
#pragma unroll
    for (int k = 0; k < C; k++) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            wv[k][j] = 1.0f;
            aw[k][j] = ab[k][j] = 0.0f;
        }
        const int c = (k * lanes + l) * 8;
        if (w && c < N) load8_rt(w, w_dt, RAGGED ? piece_begin(c, N) : c, N, wv[k]);
    }
    for (int64_t i = 0; i < rounds; i++, row += step) {
        if (kLean) load(row);
        float h[C][8], t[C][8], st[H], sth[H];
#pragma unroll
        for (int k = 0; k < H; k++) st[k] = sth[k] = 0.0f;
#pragma unroll
        for (int k = 0; k < C; k++) {
            raw8_to_f32<DT>(rx[k], h[k]);
            raw8_to_f32<DT>(rg[k], t[k]);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                h[k][j] = (h[k][j] - mean) * rstd;
                if (SUMS) {
                    aw[k][j] = fmaf(t[k][j], h[k][j], aw[k][j]);
                    ab[k][j] += t[k][j];
                }
                t[k][j] *= wv[k][j];  // zeros past the row: they add nothing to any sum
                const float own = !RAGGED || own_element((k * lanes + l) * 8, N, j) ? t[k][j] : 0.0f;
                st[k % H] += own;
                sth[k % H] = fmaf(own, h[k][j], sth[k % H]);
            }
        }
        const float rs = rstd;
        if (!kLean && i + 1 < rounds) load(row + step);
        if (dx) {
            float mt, mth;
            if (L != kBlock) {
                mt = row_sum<L>(st[0], nullptr) * inv_n;
                mth = row_sum<L>(sth[0], nullptr) * inv_n;
            } else {  // both sums behind one barrier; the buffers alternate from row to row
                float *ra = red[2 * (i & 1)], *rb = red[2 * (i & 1) + 1];
                if (H == 2) {
                    const float s = four_wave_sums(st[0], st[H - 1], sth[0], sth[H - 1]);
                    float* to = threadIdx.x & 32 ? rb : ra;
                    if ((threadIdx.x & 15) == 0) to[(threadIdx.x + (threadIdx.x & 16 ? lanes : 0)) >> 6] = s;
                } else {
                    st[0] = cluster_sum<64>(st[0]);
                    sth[0] = cluster_sum<64>(sth[0]);
                    if ((threadIdx.x & 63) == 0) {
                        ra[threadIdx.x >> 6] = st[0];
                        rb[threadIdx.x >> 6] = sth[0];
                    }
                }
                __syncthreads();
                mt = cluster_sum<16>(ra[threadIdx.x & 15]) * inv_n;
                mth = cluster_sum<16>(rb[threadIdx.x & 15]) * inv_n;
            }
            if (row < M) {
#pragma unroll
                for (int k = 0; k < C; k++) {
                    const int c = (k * lanes + l) * 8;
                    if (c >= N) continue;
#pragma unroll
                    for (int j = 0; j < 8; j++) t[k][j] = (t[k][j] - fmaf(h[k][j], mth, mt)) * rs;
                    store8<DT>(elem_at<DT>(dx, row * N + (RAGGED ? piece_begin(c, N) : c)), RAGGED ? N : 8, t[k]);
                }
            }
        }
    }
    if (SUMS) {
        const bool alone = gridDim.x == 1;
        if (!kShared) {
#pragma unroll
            for (int k = 0; k < C; k++) {
                const int c = (k * lanes + l) * 8;
                if (c >= N) continue;
                const int at = RAGGED ? piece_begin(c, N) : c;
                if (alone) {
                    if (dw) store8_rt(dw, w_dt, at, N, aw[k]);
                    if (db) store8_rt(db, w_dt, at, N, ab[k]);
                } else {
                    if (dw) store8<kF32>(pw + blockIdx.x * (int64_t)N + at, N - at, aw[k]);
                    if (db) store8<kF32>(pb + blockIdx.x * (int64_t)N + at, N - at, ab[k]);
                }
            }
        } else {
#pragma unroll
            for (int which = 0; which < 2; which++) {
                void* out = which == 0 ? dw : db;
                float* part = which == 0 ? pw : pb;
                if (!out) continue;
                __syncthreads();
#pragma unroll
                for (int k = 0; k < C; k++) {
                    const int c = (k * lanes + l) * 8, at = RAGGED && c < N ? piece_begin(c, N) : c;
#pragma unroll
                    for (int j = 0; j < 8; j++) cols[kShared ? r : 0][kShared ? at + j : 0] = which == 0 ? aw[k][j] : ab[k][j];
                }
                __syncthreads();
                for (int c = threadIdx.x; c < N; c += 256) {
                    float s = cols[0][kShared ? c : 0];
                    for (int k = 1; k < R; k++) s += cols[kShared ? k : 0][kShared ? c : 0];
                    if (alone) store_rt(out, w_dt, c, s);
                    else part[blockIdx.x * (int64_t)N + c] = s;
                }
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ rows of any length
// One block per row, the row read once per pass.  1024 threads, so that the rows in work at a time stay in the L2 for the second
// and third pass (1677 x 20000 fp32: 72 us; with 256 threads, four times the rows, 101).  The sums of dw and db are a kernel of
// their own there, which reads x and dy again.
constexpr int kLongThreads = 1024;
template <int DT>
__global__ __launch_bounds__(kLongThreads) void k_ln_fwd_long(const void* __restrict__ x, int64_t x_pitch, const void* __restrict__ w,
                                                     const void* __restrict__ b, int w_dt, void* __restrict__ y,
                                                     float* __restrict__ mean_out, float* __restrict__ rstd_out, int64_t M, int64_t N,
                                                     float eps) {
    __shared__ float red[kLongThreads / 64];
    for (int64_t row = blockIdx.x; row < M; row += gridDim.x) {
        const void* xr = elem_at<DT>(x, row * x_pitch);
        float v[8], s = 0.0f;
        for (int64_t c = threadIdx.x * 8; c < N; c += kLongThreads * 8) {
            load8<DT>(elem_at<DT>(xr, c), N - c, v);
#pragma unroll
            for (int i = 0; i < 8; i++) s += v[i];
        }
        const float mean = block_sum<kLongThreads / 64>(s, red) / (float)N;
        s = 0.0f;
        for (int64_t c = threadIdx.x * 8; c < N; c += kLongThreads * 8) {
            load8<DT>(elem_at<DT>(xr, c), N - c, v);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float d = c + i < N ? v[i] - mean : 0.0f;
                s = fmaf(d, d, s);
            }
        }
        const float rstd = 1.0f / sqrtf(block_sum<kLongThreads / 64>(s, red) / (float)N + eps);
        void* yr = elem_at<DT>(y, row * N);
        for (int64_t c = threadIdx.x * 8; c < N; c += kLongThreads * 8) {
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
__global__ __launch_bounds__(kLongThreads) void k_ln_bwd_long(const void* __restrict__ dy, int64_t dy_pitch, const void* __restrict__ x,
                                                     int64_t x_pitch, const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                                                     const void* __restrict__ w, int w_dt, void* __restrict__ dx, int64_t M, int64_t N) {
    __shared__ float red[kLongThreads / 64];
    for (int64_t row = blockIdx.x; row < M; row += gridDim.x) {
        const void *xr = elem_at<DT>(x, row * x_pitch), *gr = elem_at<DT>(dy, row * dy_pitch);
        void* dr = elem_at<DT>(dx, row * N);
        const float mean = mean_in[row], rstd = rstd_in[row];
        float v[8], t[8], wv[8], st = 0.0f, sth = 0.0f;
        for (int64_t c = threadIdx.x * 8; c < N; c += kLongThreads * 8) {
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
        const float mt = block_sum<kLongThreads / 64>(st, red) / (float)N, mth = block_sum<kLongThreads / 64>(sth, red) / (float)N;
        for (int64_t c = threadIdx.x * 8; c < N; c += kLongThreads * 8) {
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
// 32 columns a block (one 128-byte line of each partial row); 32 slices of threads take the rows in turn, eight loads in flight
// each (one load at a time took 15 us more at 512 x 4096); slice sums are added in slice order.  blockIdx.y: 0 = the first pair
// given, 1 = the second; blockIdx.z: rows of blocks, as many to a row as a launch takes in one dimension.
constexpr int kSumCols = 32, kSumSlices = 32;
__global__ __launch_bounds__(kSumCols* kSumSlices) void k_ln_sum_partials(const float* __restrict__ pw, void* __restrict__ dw,
                                                                         const float* __restrict__ pb, void* __restrict__ db, int dt,
                                                                         int64_t rows, int64_t N) {
    __shared__ float red[kSumSlices][kSumCols];
    const int col = threadIdx.x % kSumCols, slice = threadIdx.x / kSumCols;
    const int64_t c = ((int64_t)blockIdx.z * gridDim.x + blockIdx.x) * kSumCols + col;
    const float* p = blockIdx.y == 0 && dw ? pw : pb;
    void* out = blockIdx.y == 0 && dw ? dw : db;
    float s = 0.0f;
    if (c < N)
        for (int64_t r0 = slice; r0 < rows; r0 += kSumSlices * 8) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int64_t r = r0 + k * kSumSlices;
                v[k] = r < rows ? p[r * N + c] : 0.0f;
            }
            s += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
        }
    red[slice][col] = s;
    __syncthreads();
    if (slice == 0 && c < N) {
        s = red[0][col];
#pragma unroll
        for (int k = 1; k < kSumSlices; k++) s += red[k][col];
        store_rt(out, dt, c, s);
    }
}

}  // namespace coat

using namespace coat;

static bool ln_dtype(int dt) { return dt == COAT_F32 || dt == COAT_BF16 || dt == COAT_F16; }
static bool ln_aligned(const void* p, int dt) { return ((uintptr_t)p & (dt == COAT_F32 ? 3u : 1u)) == 0; }

// How rows of N elements are held in registers: threads of a block, rows it works on at a time; threads 0: they are not.
struct LnShape {
    int threads, rows;
};
// sums: the kernel that also sums dw and db, which takes the longest rows with 512 threads: their sums, weights and values would
// not fit into the 128 registers that each of 1024 threads has.
static LnShape ln_shape(int64_t N, bool sums) {
    if (N <= 512) return {256, N <= 64 ? 32 : N <= 128 ? 16 : N <= 256 ? 8 : 4};
    if (N <= 8192) return {(int)((N + 511) / 512) * 64, 1};
    if (N <= COAT_LAYER_NORM_ROW) return {sums ? (int)((N + 2047) / 2048) * 64 : (int)((N + 1023) / 1024) * 64, 1};
    return {0, 1};
}
// Calls f(L, C, RAGGED) (as integral constants) for that form.
template <bool SUMS, typename F> static void ln_form(int64_t N, F f) {
#define FORM(LANES, PIECES)                                                                                                      \
    if (N % 8) f(std::integral_constant<int, LANES>(), std::integral_constant<int, PIECES>(), std::integral_constant<bool, true>()); \
    else f(std::integral_constant<int, LANES>(), std::integral_constant<int, PIECES>(), std::integral_constant<bool, false>())
    if (N <= 64) { FORM(8, 1); }
    else if (N <= 128) { FORM(16, 1); }
    else if (N <= 256) { FORM(32, 1); }
    else if (N <= 512) { FORM(64, 1); }
    else if (N <= 8192) { FORM(kBlock, 1); }
    else { FORM(kBlock, (SUMS ? 4 : 2)); }
    static_assert(COAT_LAYER_NORM_ROW == form_threads(kBlock, 4) * 4 * 8 && COAT_LAYER_NORM_ROW == form_threads(kBlock, 2) * 2 * 8, "longest rows");
#undef FORM
}
static int64_t ln_rounds(int64_t M, int64_t N) {
    const int rows = ln_shape(N, true).rows;
    return (M + rows - 1) / rows;
}
// Blocks of a kernel that only streams: 2^20 threads.
static unsigned ln_blocks(int64_t M, int64_t N, int threads) {
    const int64_t rounds = ln_rounds(M, N), most = (1 << 20) / threads;
    return (unsigned)(rounds < most ? rounds : most);
}

template <int DT>
static int ln_forward(const void* x, int64_t x_pitch, const void* w, const void* b, int w_dtype, void* y, float* mean, float* rstd,
                      int64_t M, int64_t N, float eps, hipStream_t st) {
    const LnShape shape = ln_shape(N, false);
    if (shape.threads)
        ln_form<false>(N, [&](auto lanes, auto pieces, auto ragged) {
            hipLaunchKernelGGL((k_ln_fwd<DT, decltype(lanes)::value, decltype(pieces)::value, decltype(ragged)::value>),
                               dim3(ln_blocks(M, N, shape.threads)), dim3(shape.threads), 0, st, x, x_pitch, w, b, w_dtype, y, mean, rstd, M,
                               (int)N, eps);
        });
    else
        hipLaunchKernelGGL((k_ln_fwd_long<DT>), dim3((unsigned)(M < 65536 ? M : 65536)), dim3(kLongThreads), 0, st, x, x_pitch, w, b, w_dtype, y, mean,
                           rstd, M, N, eps);
    return coat_launch_status();
}

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
    hipStream_t st = (hipStream_t)stream;
    switch (x_dtype) {
        case COAT_F32: return ln_forward<kF32>(x, x_pitch, w, b, w_dtype, y, mean, rstd, M, N, eps, st);
        case COAT_BF16: return ln_forward<kBF16>(x, x_pitch, w, b, w_dtype, y, mean, rstd, M, N, eps, st);
        default: return ln_forward<kF16>(x, x_pitch, w, b, w_dtype, y, mean, rstd, M, N, eps, st);
    }
}

extern "C" int coat_layer_norm_partials(int64_t M, int64_t N) {
    if (M < 0 || N <= 0) return COAT_EINVAL;
    // As many blocks as keep the memory busy: 256 of 512 threads and more, up to 1024 of fewer threads, whole numbers a CU (8192 x
    // 4096 bf16: 41 us with 256, 43 with 384, 49 with 1024).  With few rows, fewer: a partial row costs as much to write and to
    // sum as it saves (1024 x 4096 bf16: 14 us with 192, 23 with 1024; the factor is fitted to such sweeps).
    const int threads = ln_shape(N, true).threads ? ln_shape(N, true).threads : 256;
    // A few rows take one block, which needs no second kernel ([4, 4096] bf16: 12 us a call instead of 18).
    if (ln_shape(N, true).threads && ln_rounds(M, N) <= 8) return 1;
    const int64_t rounds = ln_rounds(M, N), per_cu = N > 8192 || threads > 960 ? 1 : 960 / threads > 4 ? 4 : 960 / threads, most = 256 * per_cu;
    const double balanced = sqrt(27.0 * (double)rounds * (N < 4096 ? 4096.0 / (double)N : 1.0));
    int64_t n = balanced < (double)most ? (int64_t)balanced : most;
    if (!ln_shape(N, true).threads) {  // the separate kernel has a block for every 2048 columns of a partial row: 1024 in all
        const int64_t strips = (N + 2047) / 2048, each = strips < 1024 ? 1024 / strips : 1;
        if (n > each) n = each;
    }
    if (n > rounds) n = rounds;
    return (int)(n < 1 ? 1 : n);
}

template <int DT>
static int ln_backward(const void* dy, int64_t dy_pitch, const void* x, int64_t x_pitch, const float* mean, const float* rstd,
                       const void* w, int w_dtype, void* dx, void* dw, void* db, int wb_dtype, float* pw, float* pb, int n_partial,
                       int64_t M, int64_t N, hipStream_t st) {
    if (n_partial > ln_rounds(M, N)) n_partial = (int)ln_rounds(M, N);
    const bool sums = dw || db;
    LnShape shape = ln_shape(N, sums);
    if (!sums && N > 8192 && shape.threads) shape.threads = 2 * ln_shape(N, true).threads;  // the same halves of a row as with the sums
    if (M > 0 && shape.threads) {
#define BACKWARD(SUMS, BLOCKS)                                                                                                           \
    ln_form<SUMS>(N, [&](auto lanes, auto pieces, auto ragged) {                                                                         \
        hipLaunchKernelGGL((k_ln_bwd<DT, decltype(lanes)::value, decltype(pieces)::value, decltype(ragged)::value, SUMS>), dim3(BLOCKS), \
                           dim3(shape.threads), 0, st, dy, dy_pitch, x, x_pitch, mean, rstd, w, w_dtype, dx, dw, db, pw, pb, M, (int)N);                                       \
    })
        if (sums) BACKWARD(true, (unsigned)n_partial);
        else BACKWARD(false, ln_blocks(M, N, shape.threads));
#undef BACKWARD
        if (const int rc = coat_launch_status()) return rc;
        if (sums && n_partial == 1) return COAT_OK;
    } else if (M > 0) {
        if (dx) {
            hipLaunchKernelGGL((k_ln_bwd_long<DT>), dim3((unsigned)(M < 65536 ? M : 65536)), dim3(kLongThreads), 0, st, dy, dy_pitch, x, x_pitch, mean,
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
        constexpr int64_t kRow = coat_max_blocks(kSumCols * kSumSlices);
        const int64_t blocks = (N + kSumCols - 1) / kSumCols;
        const dim3 grid((unsigned)(blocks < kRow ? blocks : kRow), dw && db ? 2 : 1, (unsigned)((blocks + kRow - 1) / kRow));
        hipLaunchKernelGGL(k_ln_sum_partials, grid, dim3(kSumCols * kSumSlices), 0, st, pw, dw, pb, db, wb_dtype, rows, N);
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
    const bool one_block = n_partial == 1 && ln_shape(N, true).threads;  // writes the sums themselves
    if ((dw || db) && M > 0 && ((!partial && !one_block) || n_partial < 1 || n_partial > 65535)) return COAT_EINVAL;
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
