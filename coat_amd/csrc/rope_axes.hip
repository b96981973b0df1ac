// Rotary positions with several axes (time, height, width, ...), q and k in one launch, forward and backward, beside the
// one-axis rotary of rope.hip.
//
//   q, k [batch, seq, heads, head_dim]; pos int64 [axes, batch, seq]; pair j of `pairs` (2 * pairs <= head_dim) turns by
//   pos[axis[j]] * turns[j] whole turns (turns = frequency / 2 pi);
//   y1 = x1 cos - x2 sin, y2 = x2 cos + x1 sin on the elements (j, j + pairs), or (2 j, 2 j + 1) with `adjacent`;
//   elements from 2 * pairs on are copied; inverse: the negated angle, which is the backward pass.
// The angle is reduced to a fraction of a turn in 64 bits: in fp32 a position of 10^5 would be off by 6e-3 radians before the
// sine is taken.  Sine and cosine are fp32, the rotation fp32, rounded once to the tensor's type.
//
// A block takes a few tokens: its threads first compute the sines and cosines of those tokens into LDS, once for all heads of q
// and k (computing them per head would cost more arithmetic than the stream takes time), then stream the heads.  No tables of
// positions in memory: the positions may be anything, and a token's angles cost 8 bytes an axis to read.
#include <math.h>

#include "coat_host.h"
#include "elem_io.h"

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
    float sign;
};

template <int DT, bool ADJ>
__global__ __launch_bounds__(256) void k_rope_axes(RopeArgs A) {
    __shared__ float2 cs[kRopeSlots];
    const int64_t first = (int64_t)blockIdx.x * A.per_block;
    const int here = (int)(A.tokens - first < A.per_block ? A.tokens - first : A.per_block);
    for (int i = threadIdx.x; i < here * A.pairs; i += 256) {
        const int t = i / A.pairs, j = i - t * A.pairs;
        const int64_t token = first + t, b = token / A.seq, s = token - b * A.seq;
        const int a = min(max(A.axis[j], 0), A.axes - 1);
        const double turns = (double)A.pos[a * A.pos_sa + b * A.pos_sb + s * A.pos_ss] * A.turns[j];
        float sn, c;
        sincospif(2.0f * (float)(turns - rint(turns)), &sn, &c);
        cs[i] = make_float2(c, A.sign * sn);
    }
    __syncthreads();
    // a job is one 8-element piece: of the first halves together with the same piece of the second halves, of adjacent pairs,
    // or of the rest behind the pairs
    const int rot = 2 * A.pairs, heads = A.q.heads + A.k.heads;
    const int turning = ((ADJ ? rot : A.pairs) + 7) >> 3, pieces = turning + ((A.head_dim - rot + 7) >> 3);
    const int jobs = here * heads * pieces;
    for (int job = threadIdx.x; job < jobs; job += 256) {
        const int th = job / pieces, piece = job - th * pieces, t = th / heads;
        int head = th - t * heads;
        const int64_t token = first + t, b = token / A.seq, s = token - b * A.seq;
        const bool is_k = head >= A.q.heads;
        const RopeTensor& T = is_k ? A.k : A.q;
        if (is_k) head -= A.q.heads;
        const void* x = elem_at<DT>(T.x, b * T.sb + s * T.ss + head * T.sh);
        void* y = elem_at<DT>(T.y, (token * T.heads + head) * A.head_dim);
        float u[8], v[8];
        if (piece >= turning) {
            const int e = rot + (piece - turning) * 8;
            load8<DT>(elem_at<DT>(x, e), A.head_dim - e, u);
            store8<DT>(elem_at<DT>(y, e), A.head_dim - e, u);
        } else if (ADJ) {
            const int e = piece * 8;
            load8<DT>(elem_at<DT>(x, e), rot - e, u);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float2 c = cs[t * A.pairs + min((e >> 1) + i, A.pairs - 1)];
                v[2 * i] = u[2 * i] * c.x - u[2 * i + 1] * c.y;
                v[2 * i + 1] = u[2 * i + 1] * c.x + u[2 * i] * c.y;
            }
            store8<DT>(elem_at<DT>(y, e), rot - e, v);
        } else {
            const int e = piece * 8;
            load8<DT>(elem_at<DT>(x, e), A.pairs - e, u);
            load8<DT>(elem_at<DT>(x, e + A.pairs), A.pairs - e, v);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float2 c = cs[t * A.pairs + min(e + i, A.pairs - 1)];
                const float x1 = u[i], x2 = v[i];
                u[i] = x1 * c.x - x2 * c.y;
                v[i] = x2 * c.x + x1 * c.y;
            }
            store8<DT>(elem_at<DT>(y, e), A.pairs - e, u);
            store8<DT>(elem_at<DT>(y, e + A.pairs), A.pairs - e, v);
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
    if (2 * (int64_t)pairs > head_dim || q_heads > 4096 || k_heads > 4096 || head_dim > 2 * kRopeSlots) return COAT_ESHAPE;
    if (batch == 0 || seq == 0 || q_heads + k_heads == 0) return COAT_OK;
    if ((q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out)) || !pos || !turns || !axis) return COAT_EINVAL;
    const uintptr_t mask = dtype == COAT_F32 ? 3 : 1;
    if ((((uintptr_t)q | (uintptr_t)q_out | (uintptr_t)k | (uintptr_t)k_out) & mask) || (((uintptr_t)pos | (uintptr_t)turns) & 7) ||
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
    int per = 4;
    while (per > 1 && per * pairs > kRopeSlots) per >>= 1;
    A.per_block = per;
    const int64_t blocks = (A.tokens + per - 1) / per;
    if (blocks > 0x7fffffffll) return COAT_ESHAPE;
    const dim3 grid((unsigned)blocks);
    hipStream_t st = (hipStream_t)stream;
#define ROPE(DT)                                                                                  \
    if (adjacent) hipLaunchKernelGGL((k_rope_axes<DT, true>), grid, dim3(256), 0, st, A);         \
    else hipLaunchKernelGGL((k_rope_axes<DT, false>), grid, dim3(256), 0, st, A)
    if (dtype == COAT_F32) { ROPE(kF32); }
    else if (dtype == COAT_BF16) { ROPE(kBF16); }
    else { ROPE(kF16); }
#undef ROPE
    return coat_launch_status();
}
