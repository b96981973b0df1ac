// Rotary positions with several axes (time, height, width, ...), q and k in one launch, forward and backward, beside the
// one-axis rotary of rope.hip.
//
//   q, k [batch, seq, heads, head_dim]; pos int64 [axes, batch, seq]; pair j of `pairs` (2 * pairs <= head_dim) turns by
//   pos[axis[j]] * turns[j] whole turns (turns = frequency / 2 pi);
//   y1 = x1 cos - x2 sin, y2 = x2 cos + x1 sin on the elements (j, j + pairs), or (2 j, 2 j + 1) with `adjacent`;
//   elements from 2 * pairs on are copied; inverse: the negated angle, which is the backward pass.
// The angle is reduced to a fraction of a turn in 64 bits: in fp32 a position of 10^5 would be off by 6e-3 radians before the
// sine is taken.  Sine and cosine are fp32, for fp32 tensors with what the rounded fraction lost added back (in the mean square
// they are off by 4.5e-8 of their size so, by 5.7e-8 without); the rotation is fp32, rounded once to the tensor's type.
//
// A block takes a few tokens: its threads first compute the sines and cosines of those tokens into LDS, once for all heads of q
// and k (computing them per head would cost more arithmetic than the stream takes time), then stream the heads.  No tables of
// positions in memory: the positions may be anything, and a token's angles cost 8 bytes an axis to read.
#include <math.h>

#include "coat_host.h"
#include "elem_io.h"
#include "tensor_list.h"

namespace coat {

constexpr int kRopeSlots = 1024;  // (token, pair) slots of a block: 8 KB of LDS

struct RopeTensor {
    const void* x;
    void* y;
    int64_t sb, ss, sh;  // strides of x in elements; y is dense
    int heads;
};
struct RopeArgs {
    RopeTensor q, k;
    const int64_t* pos;
    int64_t pos_sa, pos_sb, pos_ss;
    const double* turns;
    const int32_t* axis;
    int64_t tokens, seq;
    int axes, head_dim, pairs, per_block;  // per_block: tokens a block takes at a time
    uint32_t magic_pieces, magic_heads, magic_pairs;
    float sign;
};

// n / d for n * d < 2^32, with m = ceil(2^32 / d)
__device__ __forceinline__ uint32_t div_magic(uint32_t n, uint32_t d, uint32_t m) { return d == 1 ? n : __umulhi(n, m); }

// WHOLE: pairs and the rest are multiples of 8.
template <int DT, bool ADJ, bool WHOLE>
__global__ __launch_bounds__(256) void k_rope_axes(RopeArgs A) {
    __shared__ float2 cs[kRopeSlots];
    // rows of blocks, as many to a row as a launch takes in one dimension; in the last row blocks may have no tokens left (a branch around
    // the rest for them cost 1 % at 4 x 2048 tokens)
    const int64_t first = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * A.per_block;
    const int64_t left_over = A.tokens - first;
    const int here = left_over <= 0 ? 0 : left_over < A.per_block ? (int)left_over : A.per_block;
    // a job is one 8-element piece: of the first halves together with the same piece of the second halves, of adjacent pairs,
    // or of the rest behind the pairs
    const int rot = 2 * A.pairs, heads = A.q.heads + A.k.heads;
    const int turning = ((ADJ ? rot : A.pairs) + 7) >> 3, pieces = turning + ((A.head_dim - rot + 7) >> 3);
    const int jobs = here * heads * pieces;
    struct Job {
        Raw8<DT> a, b;
        void* y;
        int piece, token, e, n;
    };
    auto fetch = [&](int job) {
        Job J;
        const uint32_t th = div_magic(job, pieces, A.magic_pieces);
        J.piece = job - (int)th * pieces;
        J.token = div_magic(th, heads, A.magic_heads);
        int head = (int)th - J.token * heads;
        const int64_t token = first + J.token, b = token / A.seq, s = token - b * A.seq;
        const bool is_k = head >= A.q.heads;
        if (is_k) head -= A.q.heads;
        const void* x = is_k ? elem_at<DT>(A.k.x, b * A.k.sb + s * A.k.ss + head * A.k.sh)
                             : elem_at<DT>(A.q.x, b * A.q.sb + s * A.q.ss + head * A.q.sh);
        J.y = is_k ? elem_at<DT>(A.k.y, (token * A.k.heads + head) * A.head_dim) : elem_at<DT>(A.q.y, (token * A.q.heads + head) * A.head_dim);
        // the run of elements that the piece belongs to (all pairs, the first and second halves, or the rest), and its place there
        const bool rest = J.piece >= turning;
        J.e = (rest ? J.piece - turning : J.piece) * 8;
        J.n = rest ? A.head_dim - rot : ADJ ? rot : A.pairs;
        J.a = load_piece<DT, !WHOLE, true>(rest ? elem_at<DT>(x, rot) : x, J.e, J.n);
        if (!ADJ && !rest) J.b = load_piece<DT, !WHOLE, true>(elem_at<DT>(x, A.pairs), J.e, J.n);
        if (!WHOLE) J.e = piece_begin(J.e, J.n);
        return J;
    };
    Job J;
    if ((int)threadIdx.x < jobs) J = fetch(threadIdx.x);  // in flight while the sines are computed
    for (int i = threadIdx.x; i < here * A.pairs; i += 256) {
        const int t = div_magic(i, A.pairs, A.magic_pairs), j = i - t * A.pairs;
        const int64_t token = first + t, b = token / A.seq, s = token - b * A.seq;
        const int a = min(max(A.axis[j], 0), A.axes - 1);
        const double turns = (double)A.pos[a * A.pos_sa + b * A.pos_sb + s * A.pos_ss] * A.turns[j];
        const double part = turns - rint(turns);
        const float rounded = (float)part;
        float sn, c;
        sincospif(2.0f * rounded, &sn, &c);
        if (DT == kF32) {  // what the argument lost (up to 9e-8 radians; 16-bit tensors do not show it), to first order
            const float lost = 6.28318531f * (float)(part - (double)rounded), s0 = sn;
            sn = fmaf(lost, c, sn);
            c = fmaf(-lost, s0, c);
        }
        cs[i] = make_float2(c, A.sign * sn);
    }
    __syncthreads();
    for (int job = threadIdx.x; job < jobs;) {
        const int e = J.e, left = WHOLE ? 8 : J.n, piece = J.piece;  // fewer than 8 only where the whole run is
        void* y = J.y;
        const float2* c = cs + J.token * A.pairs;
        float u[8], v[8];
        raw8_to_f32<DT>(J.a, u);
        if (!ADJ) raw8_to_f32<DT>(J.b, v);
        job += 256;
        if (job < jobs) J = fetch(job);
        if (piece >= turning) {
            store8<DT>(elem_at<DT>(y, rot + e), left, u);
        } else if (ADJ) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float2 f = c[WHOLE ? (e >> 1) + i : min((e >> 1) + i, A.pairs - 1)];
                v[2 * i] = u[2 * i] * f.x - u[2 * i + 1] * f.y;
                v[2 * i + 1] = u[2 * i + 1] * f.x + u[2 * i] * f.y;
            }
            store8<DT>(elem_at<DT>(y, e), left, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float2 f = c[WHOLE ? e + i : min(e + i, A.pairs - 1)];
                const float x1 = u[i], x2 = v[i];
                u[i] = x1 * f.x - x2 * f.y;
                v[i] = x2 * f.x + x1 * f.y;
            }
            store8<DT>(elem_at<DT>(y, e), left, u);
            store8<DT>(elem_at<DT>(y, e + A.pairs), left, v);
        }
    }
}

}  // namespace coat

using namespace coat;

extern "C" int coat_rope_axes(const void* q, void* q_out, int64_t q_sb, int64_t q_ss, int64_t q_sh, int q_heads, const void* k,
                              void* k_out, int64_t k_sb, int64_t k_ss, int64_t k_sh, int k_heads, int dtype, const int64_t* pos,
                              int64_t pos_sa, int64_t pos_sb, int64_t pos_ss, int axes, const double* turns, const int32_t* axis,
                              int pairs, int head_dim, int adjacent, int inverse, int64_t batch, int64_t seq, void* stream) {
    if (dtype != COAT_F32 && dtype != COAT_BF16 && dtype != COAT_F16) return COAT_EDTYPE;
    if (batch < 0 || seq < 0 || q_heads < 0 || k_heads < 0 || axes < 1 || pairs < 1 || head_dim < 2 || adjacent < 0 || adjacent > 1 ||
        inverse < 0 || inverse > 1)
        return COAT_EINVAL;
    if (2 * (int64_t)pairs > head_dim || q_heads > 1024 || k_heads > 1024 || head_dim > 2 * kRopeSlots) return COAT_ESHAPE;
    if (batch == 0 || seq == 0 || q_heads + k_heads == 0) return COAT_OK;
    if (batch > ((int64_t)1 << 40) / seq) return COAT_ESHAPE;
    if ((q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out)) || !pos || !turns || !axis) return COAT_EINVAL;
    const uintptr_t mask = dtype == COAT_F32 ? 3 : 1, at_q = (uintptr_t)q | (uintptr_t)q_out, at_k = (uintptr_t)k | (uintptr_t)k_out;
    if ((q_heads && (at_q & mask)) || (k_heads && (at_k & mask)) || (((uintptr_t)pos | (uintptr_t)turns) & 7) ||
        ((uintptr_t)axis & 3))
        return COAT_EALIGN;
    RopeArgs A;
    A.q = RopeTensor{q, q_out, q_sb, q_ss, q_sh, q_heads};
    A.k = RopeTensor{k, k_out, k_sb, k_ss, k_sh, k_heads};
    A.pos = pos;
    A.pos_sa = pos_sa; A.pos_sb = pos_sb; A.pos_ss = pos_ss;
    A.turns = turns;
    A.axis = axis;
    A.tokens = batch * seq;
    A.seq = seq;
    A.axes = axes; A.head_dim = head_dim; A.pairs = pairs;
    A.sign = inverse ? -1.0f : 1.0f;
    const int turning = ((adjacent ? 2 * pairs : pairs) + 7) / 8, pieces = turning + (head_dim - 2 * pairs + 7) / 8;
    auto magic = [](int d) { return (uint32_t)((((uint64_t)1 << 32) + d - 1) / d); };
    A.magic_pieces = magic(pieces);
    A.magic_heads = magic(q_heads + k_heads);
    A.magic_pairs = magic(pairs);
    const bool whole = head_dim % 8 == 0 && (adjacent ? pairs % 4 == 0 : pairs % 8 == 0);
    // about 512 pieces a block: two rounds of its 256 threads, the second in flight under the first, next to the sines of as few
    // tokens as possible (bf16, 4 x 2048 tokens, 64 heads of 128: one token 46 us, four 48, sixteen 69; 4 x 4096 tokens, 16 heads
    // of 64: one 22 us, eight 13); fewer where the tokens are too few to fill the card.
    const int64_t per_token = (int64_t)(q_heads + k_heads) * pieces;
    int per = 1;
    while (per < 16 && 2 * per * per_token <= 768 && 2 * per * pairs <= kRopeSlots && A.tokens / (2 * per) >= 512) per *= 2;
    A.per_block = per;
    const int64_t blocks = (A.tokens + per - 1) / per;
    if (blocks > 0x7fffffffll) return COAT_ESHAPE;
    constexpr int64_t kRow = coat_max_blocks(256);
    const dim3 grid((unsigned)(blocks < kRow ? blocks : kRow), (unsigned)((blocks + kRow - 1) / kRow));
    hipStream_t st = (hipStream_t)stream;
#define ROPE(DT)                                                                                                    \
    if (adjacent && whole) hipLaunchKernelGGL((k_rope_axes<DT, true, true>), grid, dim3(256), 0, st, A);             \
    else if (adjacent) hipLaunchKernelGGL((k_rope_axes<DT, true, false>), grid, dim3(256), 0, st, A);                \
    else if (whole) hipLaunchKernelGGL((k_rope_axes<DT, false, true>), grid, dim3(256), 0, st, A);                   \
    else hipLaunchKernelGGL((k_rope_axes<DT, false, false>), grid, dim3(256), 0, st, A)
    if (dtype == COAT_F32) { ROPE(kF32); }
    else if (dtype == COAT_BF16) { ROPE(kBF16); }
    else { ROPE(kF16); }
#undef ROPE
    return coat_launch_status();
}
