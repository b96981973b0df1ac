// AdamW over many tensors with both moments in fp32, and the global 2-norm of many gradient tensors that clips it, beside the
// FP8-state steps of adamw.hip.
//
//   n = sqrt(sum over all tensors of g^2);   s = min(1, max_norm / (n + 1e-6))
//   g' = s g;   m = beta1 m + (1 - beta1) g';   v = beta2 v + (1 - beta2) g'^2
//   p = p - lr (m / ((sqrt(v) / c2 + eps) c1) + wd p),   c1 = 1 - beta1^step,  c2 = sqrt(1 - beta2^step)
// the order of operations of the FP8-state steps.  p is the fp32 master copy where there is one; the parameter of 16 bits is
// then its rounding.  Everything is fp32; the sum of squares is taken in 64 bits (squares of fp32 gradients neither overflow
// nor lose small tensors next to large ones, and the order of the additions no longer shows), in a fixed order: no atomics.
//
// Both kernels stream.  The records of the tensors travel in the kernel arguments (4 KB): no copy to the device ahead of the
// launch, nothing that a captured graph would have to keep alive.
#include <math.h>

#include <memory>
#include <new>

#include "coat_host.h"
#include "elem_io.h"
#include "tensor_list.h"

namespace coat {

// ------------------------------------------------------------------------------------------------ sum of squares
constexpr int kNormMax = 184;        // tensors per launch: what the 4 KB of kernel arguments hold
constexpr int kNormChunk = 8192;     // elements a block takes at a time
constexpr int kNormBlocks = 2048;    // blocks (partial sums) per launch at most
struct NormArgs {
    const void* g[kNormMax];
    int64_t numel[kNormMax];
    uint32_t first_chunk[kNormMax + 1];  // first_chunk[count] = number of chunks
    uint8_t dt[kNormMax];
    int count;
};

// Index of the last tensor whose first chunk is not after `chunk` (wave-uniform).
__device__ __forceinline__ int find_tensor(const uint32_t* first, int count, uint32_t chunk) {
    int lo = 0, hi = count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (chunk >= first[mid]) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// 16 bytes a lane and load, all loads of a chunk in flight, non-temporal: the gradients are read once here, and the step that reads
// them again comes after all of them (1.33 GB of fp32: 250 us with ordinary loads of 32 bytes a lane, 219 with 16, 195 so).
template <int DT> __device__ __forceinline__ double sumsq_chunk(const void* g, int64_t begin, int64_t numel) {
    constexpr int E = DT == kF32 ? 4 : 8, J = kNormChunk / (256 * E);  // elements of a load, loads
    uint32_t w[J][4];
    double s = 0.0;
    if (begin + kNormChunk <= numel) {
#pragma unroll
        for (int j = 0; j < J; j++) {
            const void* p = elem_at<DT>(g, begin + (j * 256 + threadIdx.x) * E);
            if (DT == kF32) {
                const coat_u4_at4 v = __builtin_nontemporal_load((const coat_u4_at4*)p);
                w[j][0] = v.x; w[j][1] = v.y; w[j][2] = v.z; w[j][3] = v.w;
            } else {
                const coat_u4_at2 v = __builtin_nontemporal_load((const coat_u4_at2*)p);
                w[j][0] = v.x; w[j][1] = v.y; w[j][2] = v.z; w[j][3] = v.w;
            }
        }
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const double a = DT == kF32 ? u2f(w[j][k]) : elem_lo<DT>(w[j][k]), b = DT == kF32 ? 0.0f : elem_hi<DT>(w[j][k]);
                s = fma(a, a, s);
                if (DT != kF32) s = fma(b, b, s);
            }
    } else {  // the tensor's last chunk
        const int n = (int)(numel - begin);
        const void* p = elem_at<DT>(g, begin);
        Raw8<DT> r[kNormChunk / 2048];
#pragma unroll
        for (int j = 0; j < kNormChunk / 2048; j++) r[j] = load_piece<DT, true, true>(p, j * 2048 + threadIdx.x * 8, n);
#pragma unroll
        for (int j = 0; j < kNormChunk / 2048; j++) {
            const int c = j * 2048 + threadIdx.x * 8;
            float v[8];
            raw8_to_f32<DT>(r[j], v);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const double a = c < n && own_element(c, n, i) ? v[i] : 0.0f;
                s = fma(a, a, s);
            }
        }
    }
    return s;
}

__device__ __forceinline__ double block_sum_f64(double s, double* red) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    s = red[0];
    for (int k = 1; k < (int)(blockDim.x >> 6); k++) s += red[k];
    return s;
}

__global__ __launch_bounds__(256) void k_grad_sumsq(NormArgs A, double* __restrict__ partial) {
    __shared__ double red[4];
    double s = 0.0;
    const uint32_t chunks = A.first_chunk[A.count];
    for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int t = find_tensor(A.first_chunk, A.count, c);
        const int64_t begin = (int64_t)(c - A.first_chunk[t]) * kNormChunk;
        if (A.dt[t] == kF32) s += sumsq_chunk<kF32>(A.g[t], begin, A.numel[t]);
        else if (A.dt[t] == kBF16) s += sumsq_chunk<kBF16>(A.g[t], begin, A.numel[t]);
        else s += sumsq_chunk<kF16>(A.g[t], begin, A.numel[t]);
    }
    s = block_sum_f64(s, red);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// out[0] = the norm, out[1] = the factor of the gradients.  A norm that is not a number gives a factor that is not one.
__global__ __launch_bounds__(1024) void k_grad_norm(const double* __restrict__ partial, int64_t n, float max_norm, float* __restrict__ out) {
    __shared__ double red[16];
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 1024) s += partial[i];
    s = block_sum_f64(s, red);
    if (threadIdx.x == 0) {
        const double norm = sqrt(s), f = (double)max_norm / (norm + 1e-6);
        out[0] = (float)norm;
        out[1] = f > 1.0 ? 1.0f : (float)f;
    }
}

// ------------------------------------------------------------------------------------------------ the step
constexpr int kStepMax = 76;        // tensors per launch: what the 4 KB of kernel arguments hold
constexpr int kStepChunk = 1024;    // elements a block steps
constexpr int64_t kStepBlocks = coat_max_blocks(256);  // per launch
constexpr int64_t kNormChunks = 0x7fffffff;            // per launch: their numbers are 32-bit
struct Step32Tensor {
    void* p;
    const void* g;
    float *m, *v, *master;
    int64_t numel;
};
struct Step32Args {
    Step32Tensor t[kStepMax];
    uint32_t first_chunk[kStepMax + 1];
    int count;
    const float* grad_scale;
};
struct Hyper32 {
    float beta1, one_minus_beta1, beta2, one_minus_beta2, lr, wd, eps, c1, inv_c2;
};

static_assert(sizeof(NormArgs) + sizeof(double*) <= 4096 && sizeof(Step32Args) + sizeof(Hyper32) <= 4096, "kernel arguments");

// One load of each stream a thread, and short blocks: the card holds enough of them to keep the memory busy (fp32, 333 M elements:
// 1679 us or 5.56 TB/s; 2048 elements a block 1700, 4096 1736; non-temporal loads 1860).  The blocks go through the tensors from
// the end, where the norm kernel before left off.
template <int PDT, int GDT, bool MASTER>
__global__ __launch_bounds__(256) void k_adamw32(Step32Args A, Hyper32 H) {
    const uint32_t chunk = gridDim.x - 1 - blockIdx.x;
    const int ti = find_tensor(A.first_chunk, A.count, chunk);
    const Step32Tensor T = A.t[ti];
    const float gs = A.grad_scale ? *A.grad_scale : 1.0f;
    const int64_t e = (int64_t)(chunk - A.first_chunk[ti]) * kStepChunk + threadIdx.x * 4, left = T.numel - e;
    float p[4], g[4], m[4], v[4];
    if (MASTER) load4<kF32>(T.master + e, left, p);
    else load4<PDT>(elem_at<PDT>(T.p, e), left, p);
    load4<GDT>(elem_at<GDT>(T.g, e), left, g);
    load4<kF32>(T.m + e, left, m);
    load4<kF32>(T.v + e, left, v);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float gr = g[i] * gs;
        m[i] = fmaf(H.beta1, m[i], H.one_minus_beta1 * gr);
        v[i] = fmaf(H.beta2, v[i], (H.one_minus_beta2 * gr) * gr);
        const float denom = fmaf(sqrtf(v[i]), H.inv_c2, H.eps) * H.c1;
        const float update = fmaf(H.wd, p[i], m[i] / denom);
        p[i] = fmaf(-H.lr, update, p[i]);
    }
    store4<kF32>(T.m + e, left, m);
    store4<kF32>(T.v + e, left, v);
    if (MASTER) store4<kF32>(T.master + e, left, p);
    store4<PDT>(elem_at<PDT>(T.p, e), left, p);
}

}  // namespace coat

using namespace coat;

static bool opt_dtype(int dt) { return dt == COAT_F32 || dt == COAT_BF16 || dt == COAT_F16; }
static bool elem_aligned(const void* p, int dt) { return ((uintptr_t)p & (dt == COAT_F32 ? 3u : 1u)) == 0; }
static int64_t norm_chunks(int64_t numel) { return (numel + kNormChunk - 1) / kNormChunk; }

extern "C" int coat_grad_norm_partials(int count, const int64_t* numel) {
    if (count < 0 || (count > 0 && !numel)) return COAT_EINVAL;
    int64_t total = 0;
    for (int i = 0; i < count; i++)
        if (numel[i] < 0) return COAT_EINVAL;
    const int rc = coat_for_each_launch(count, numel, kNormChunk, kNormMax, kNormChunks, [&](int, int, int64_t chunks) {
        total += chunks < kNormBlocks ? chunks : kNormBlocks;
        return total > 0x7fffffff ? COAT_ESHAPE : COAT_OK;
    });
    return rc != COAT_OK ? rc : (int)total;
}

extern "C" int coat_grad_norm_multi(int count, const void* const* grads, const int* dtypes, const int64_t* numel, float max_norm,
                                    double* partial, int n_partial, float* out, void* stream) {
    const int need = coat_grad_norm_partials(count, numel);
    if (need < 0) return need;
    if ((count > 0 && (!grads || !dtypes)) || !out || !(max_norm >= 0.0f)) return COAT_EINVAL;
    if (need > 0 && (!partial || n_partial < need)) return COAT_EINVAL;
    if (((uintptr_t)partial & 7u) || !elem_aligned(out, COAT_F32)) return COAT_EALIGN;
    for (int i = 0; i < count; i++) {
        if (!opt_dtype(dtypes[i])) return COAT_EDTYPE;
        if (numel[i] == 0) continue;
        if (!grads[i]) return COAT_EINVAL;
        if (!elem_aligned(grads[i], dtypes[i])) return COAT_EALIGN;
    }
    hipStream_t st = (hipStream_t)stream;
    double* at = partial;
    const int rc = coat_for_each_launch(count, numel, kNormChunk, kNormMax, kNormChunks, [&](int first, int last, int64_t chunks) {
        NormArgs A;
        A.count = 0;
        uint32_t c = 0;
        for (int i = first; i < last; i++) {
            if (numel[i] == 0) continue;
            A.g[A.count] = grads[i];
            A.numel[A.count] = numel[i];
            A.dt[A.count] = (uint8_t)dtypes[i];
            A.first_chunk[A.count++] = c;
            c += (uint32_t)norm_chunks(numel[i]);
        }
        A.first_chunk[A.count] = c;
        const int blocks = (int)(chunks < kNormBlocks ? chunks : kNormBlocks);
        hipLaunchKernelGGL(k_grad_sumsq, dim3(blocks), dim3(256), 0, st, A, at);
        at += blocks;
        return coat_launch_status();
    });
    if (rc != COAT_OK) return rc;
    hipLaunchKernelGGL(k_grad_norm, dim3(1), dim3(1024), 0, st, partial, (int64_t)need, max_norm, out);
    return coat_launch_status();
}

extern "C" int coat_adamw_step_multi(int count, void* const* params, int p_dtype, const void* const* grads, int g_dtype,
                                     float* const* exp_avg, float* const* exp_avg_sq, float* const* masters, const int64_t* numel,
                                     const double* hyper, int step, const float* grad_scale, void* stream) {
    if (count < 0) return COAT_EINVAL;
    if (count == 0) return COAT_OK;
    if (!params || !grads || !exp_avg || !exp_avg_sq || !numel || !hyper || step < 1) return COAT_EINVAL;
    if (!opt_dtype(p_dtype) || (g_dtype != p_dtype && g_dtype != COAT_F32) || (masters && p_dtype == COAT_F32)) return COAT_EDTYPE;
    if (!(hyper[0] >= 0.0 && hyper[0] < 1.0) || !(hyper[1] >= 0.0 && hyper[1] < 1.0)) return COAT_EINVAL;
    if (!elem_aligned(grad_scale, COAT_F32)) return COAT_EALIGN;
    for (int i = 0; i < count; i++) {  // everything is checked before the first launch
        if (numel[i] < 0) return COAT_EINVAL;
        if (numel[i] > kStepBlocks * kStepChunk) return COAT_ESHAPE;
        if (numel[i] == 0) continue;
        if (!params[i] || !grads[i] || !exp_avg[i] || !exp_avg_sq[i] || (masters && !masters[i])) return COAT_EINVAL;
        if (!elem_aligned(params[i], p_dtype) || !elem_aligned(grads[i], g_dtype) || !elem_aligned(exp_avg[i], COAT_F32) ||
            !elem_aligned(exp_avg_sq[i], COAT_F32) || (masters && !elem_aligned(masters[i], COAT_F32)))
            return COAT_EALIGN;
    }
    // over all launches: a later one would read what an earlier one has stepped
    CoatSpan few[5 * kStepMax];
    std::unique_ptr<CoatSpan[]> many;
    if (count > kStepMax) {
        many.reset(new (std::nothrow) CoatSpan[5 * (size_t)count]);
        if (!many) return (int)hipErrorOutOfMemory;
    }
    CoatSpan* spans = many ? many.get() : few;
    size_t n = 0;
    for (int i = 0; i < count; i++) {
        const uintptr_t p = (uintptr_t)params[i], g = (uintptr_t)grads[i], m = (uintptr_t)exp_avg[i], v = (uintptr_t)exp_avg_sq[i];
        const size_t size = (size_t)numel[i];
        if (size == 0) continue;
        spans[n++] = {p, p + size * (p_dtype == COAT_F32 ? 4 : 2), true};
        spans[n++] = {g, g + size * (g_dtype == COAT_F32 ? 4 : 2), false};
        spans[n++] = {m, m + size * 4, true};
        spans[n++] = {v, v + size * 4, true};
        if (masters) spans[n++] = {(uintptr_t)masters[i], (uintptr_t)masters[i] + size * 4, true};
    }
    if (coat_overlap(spans, n)) return COAT_EOVERLAP;
    // hyperparameters in double, rounded once: 1 - beta2 of a beta2 that was already rounded to fp32 is off by 1e-5 at 0.999
    const double beta1 = hyper[0], beta2 = hyper[1];
    Hyper32 H;
    H.beta1 = (float)beta1;
    H.one_minus_beta1 = (float)(1.0 - beta1);
    H.beta2 = (float)beta2;
    H.one_minus_beta2 = (float)(1.0 - beta2);
    H.lr = (float)hyper[2];
    H.wd = (float)hyper[3];
    H.eps = (float)hyper[4];
    H.c1 = (float)(1.0 - pow(beta1, (double)step));
    H.inv_c2 = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)step)));
    hipStream_t st = (hipStream_t)stream;
    return coat_for_each_launch(count, numel, kStepChunk, kStepMax, kStepBlocks, [&](int first, int last, int64_t chunks) {
        Step32Args A;
        A.count = 0;
        A.grad_scale = grad_scale;
        uint32_t c = 0;
        for (int i = first; i < last; i++) {
            if (numel[i] == 0) continue;
            A.t[A.count] = Step32Tensor{params[i], grads[i], exp_avg[i], exp_avg_sq[i], masters ? masters[i] : nullptr, numel[i]};
            A.first_chunk[A.count++] = c;
            c += (uint32_t)((numel[i] + kStepChunk - 1) / kStepChunk);
        }
        A.first_chunk[A.count] = c;
        const dim3 grid((unsigned)chunks), block(256);
#define STEP(PDT, GDT, MASTER) hipLaunchKernelGGL((k_adamw32<PDT, GDT, MASTER>), grid, block, 0, st, A, H)
        if (p_dtype == COAT_F32) STEP(kF32, kF32, false);
        else if (p_dtype == COAT_BF16) {
            if (masters) { if (g_dtype == COAT_F32) STEP(kBF16, kF32, true); else STEP(kBF16, kBF16, true); }
            else { if (g_dtype == COAT_F32) STEP(kBF16, kF32, false); else STEP(kBF16, kBF16, false); }
        } else {
            if (masters) { if (g_dtype == COAT_F32) STEP(kF16, kF32, true); else STEP(kF16, kF16, true); }
            else { if (g_dtype == COAT_F32) STEP(kF16, kF32, false); else STEP(kF16, kF16, false); }
        }
#undef STEP
        return coat_launch_status();
    });
}
