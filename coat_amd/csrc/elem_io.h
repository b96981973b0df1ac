// Wide loads and stores of 16- and 32-bit elements at any element alignment, for the kernels that take row slices, odd row
// lengths and tensors laid out one after the other without padding.  The hardware's global loads and stores need no more
// than the element's own alignment (the code objects run in unaligned access mode), so a 16-byte access that crosses a line
// costs one more line, not a loop over elements.  A row that ends inside a piece takes its last eight elements as the last piece
// (piece_begin); only rows of fewer than eight, and the ends that load8 / load4 are given, go element by element.
#pragma once
#include "coat_device.h"

namespace coat {

typedef uint32_t coat_u4_at2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t coat_u2_at2 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t coat_u4_at4 __attribute__((ext_vector_type(4), aligned(4)));

template <int DT> struct ElemBytes { static constexpr int value = DT == kF32 ? 4 : 2; };
template <int DT> __device__ __forceinline__ const void* elem_at(const void* p, int64_t i) { return (const char*)p + i * ElemBytes<DT>::value; }
template <int DT> __device__ __forceinline__ void* elem_at(void* p, int64_t i) { return (char*)p + i * ElemBytes<DT>::value; }

template <int DT> __device__ __forceinline__ float elem_lo(uint32_t w) { return DT == kBF16 ? bf16lo(w) : f16lo(w); }
template <int DT> __device__ __forceinline__ float elem_hi(uint32_t w) { return DT == kBF16 ? bf16hi(w) : f16hi(w); }
template <int DT> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    return DT == kBF16 ? pack_bf16x2(lo, hi) : (f2f16(lo) | (f2f16(hi) << 16));
}

// Eight elements as they lie in memory (16 bytes of 16-bit elements, 32 of fp32), kept packed until they are used.
template <int DT> struct Raw8 { uint32_t w[DT == kF32 ? 8 : 4]; };

// p: address of the first element; left: elements from there to the end of the row (<= 0: nothing is read, zeros).
// STREAM: non-temporal loads, for a tensor that no later kernel reads again soon.
template <int DT, bool STREAM = false> __device__ __forceinline__ Raw8<DT> load_raw8(const void* p, int64_t left) {
    Raw8<DT> r;
    if (left >= 8) {
        if (DT == kF32) {
            const coat_u4_at4* q = (const coat_u4_at4*)p;
            const coat_u4_at4 a = STREAM ? __builtin_nontemporal_load(q) : q[0], b = STREAM ? __builtin_nontemporal_load(q + 1) : q[1];
            r.w[0] = a.x; r.w[1] = a.y; r.w[2] = a.z; r.w[3] = a.w;
            r.w[DT == kF32 ? 4 : 0] = b.x; r.w[DT == kF32 ? 5 : 1] = b.y; r.w[DT == kF32 ? 6 : 2] = b.z; r.w[DT == kF32 ? 7 : 3] = b.w;
        } else {
            const coat_u4_at2 a = STREAM ? __builtin_nontemporal_load((const coat_u4_at2*)p) : *(const coat_u4_at2*)p;
            r.w[0] = a.x; r.w[1] = a.y; r.w[2] = a.z; r.w[3] = a.w;
        }
    } else if (left > 0) {  // all loads in flight together: elements past the end are read from the last one and cleared
        uint32_t e[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int64_t at = i < left ? i : left - 1;
            e[i] = DT == kF32 ? ((const uint32_t*)p)[at] : ((const uint16_t*)p)[at];
        }
#pragma unroll
        for (int i = 0; i < 8; i++) e[i] = i < left ? e[i] : 0u;
#pragma unroll
        for (int k = 0; k < (DT == kF32 ? 8 : 4); k++) r.w[k] = DT == kF32 ? e[k] : e[2 * k & 7] | e[(2 * k + 1) & 7] << 16;
    } else {
#pragma unroll
        for (int k = 0; k < (DT == kF32 ? 8 : 4); k++) r.w[k] = 0;
    }
    return r;
}
// A row of n elements in pieces of eight: the last piece of a row whose length is not a multiple of 8 is the eight elements that
// end the row, so that every piece is one wide load and one wide store.  Elements that two pieces hold are computed and stored
// twice, with the same value; sums count them in the first (own_element).  Rows of fewer than eight elements are one short piece.
// (Element-wise ends cost much more: picking single elements waits for their load at once, which holds up every row of a block.)
__device__ __forceinline__ int piece_begin(int c, int n) { return c + 8 <= n || n < 8 ? c : n - 8; }
// Whether element j of the piece at piece_begin(c, n) belongs to column c + 0 .. 7 of the row, and not to the piece before.
__device__ __forceinline__ bool own_element(int c, int n, int j) { return n >= 8 ? j >= c + 8 - n : j < n; }
// RAGGED: n need not be a multiple of 8.  Otherwise c is below n only where a whole piece is.  Zeros if not valid or past the row.
template <int DT, bool RAGGED, bool STREAM> __device__ __forceinline__ Raw8<DT> load_piece(const void* row, int c, int n, bool valid = true) {
    Raw8<DT> r;
#pragma unroll
    for (int k = 0; k < (DT == kF32 ? 8 : 4); k++) r.w[k] = 0;
    if (valid && c < n) {
        if (!RAGGED || n >= 8) r = load_raw8<DT, STREAM>(elem_at<DT>(row, RAGGED ? piece_begin(c, n) : c), 8);
        else r = load_raw8<DT>(row, n);
    }
    return r;
}
template <int DT> __device__ __forceinline__ void raw8_to_f32(const Raw8<DT>& r, float* o) {
    if (DT == kF32) {
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = u2f(r.w[DT == kF32 ? i : 0]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            o[2 * k] = elem_lo<DT>(r.w[k]);
            o[2 * k + 1] = elem_hi<DT>(r.w[k]);
        }
    }
}
template <int DT> __device__ __forceinline__ void load8(const void* p, int64_t left, float* o) { raw8_to_f32<DT>(load_raw8<DT>(p, left), o); }
template <int DT> __device__ __forceinline__ void store8(void* p, int64_t left, const float* v) {
    if (left >= 8) {
        if (DT == kF32) {
            ((coat_u4_at4*)p)[0] = (coat_u4_at4){f2u(v[0]), f2u(v[1]), f2u(v[2]), f2u(v[3])};
            ((coat_u4_at4*)p)[1] = (coat_u4_at4){f2u(v[4]), f2u(v[5]), f2u(v[6]), f2u(v[7])};
        } else {
            *(coat_u4_at2*)p = (coat_u4_at2){pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]), pack2<DT>(v[4], v[5]), pack2<DT>(v[6], v[7])};
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < left) store_from_f32<DT>(p, i, v[i]);
    }
}
// Four elements, for kernels whose widest tensors are fp32: lane l of a wave then reads bytes 16 l .. 16 l + 15 of one run with each
// load (with eight fp32 elements a lane every load touches each line twice).
template <int DT> __device__ __forceinline__ void load4(const void* p, int64_t left, float* o) {
    if (left >= 4) {
        if (DT == kF32) {
            const coat_u4_at4 a = *(const coat_u4_at4*)p;
            o[0] = u2f(a.x); o[1] = u2f(a.y); o[2] = u2f(a.z); o[3] = u2f(a.w);
        } else {
            const coat_u2_at2 a = *(const coat_u2_at2*)p;
            o[0] = elem_lo<DT>(a.x); o[1] = elem_hi<DT>(a.x); o[2] = elem_lo<DT>(a.y); o[3] = elem_hi<DT>(a.y);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = i < left ? load_as_f32<DT>(p, i) : 0.0f;
    }
}
template <int DT> __device__ __forceinline__ void store4(void* p, int64_t left, const float* v) {
    if (left >= 4) {
        if (DT == kF32) *(coat_u4_at4*)p = (coat_u4_at4){f2u(v[0]), f2u(v[1]), f2u(v[2]), f2u(v[3])};
        else *(coat_u2_at2*)p = (coat_u2_at2){pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3])};
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (i < left) store_from_f32<DT>(p, i, v[i]);
    }
}
// The same with the element type known at run time only (weights and biases): a wave-uniform branch.
__device__ __forceinline__ void load8_rt(const void* p, int dt, int64_t i, int64_t n, float* o) {
    if (dt == kF32) load8<kF32>(elem_at<kF32>(p, i), n - i, o);
    else if (dt == kBF16) load8<kBF16>(elem_at<kBF16>(p, i), n - i, o);
    else load8<kF16>(elem_at<kF16>(p, i), n - i, o);
}

__device__ __forceinline__ void store8_rt(void* p, int dt, int64_t i, int64_t n, const float* v) {
    if (dt == kF32) store8<kF32>(elem_at<kF32>(p, i), n - i, v);
    else if (dt == kBF16) store8<kBF16>(elem_at<kBF16>(p, i), n - i, v);
    else store8<kF16>(elem_at<kF16>(p, i), n - i, v);
}
__device__ __forceinline__ void store_rt(void* p, int dt, int64_t i, float v) {
    if (dt == kF32) store_from_f32<kF32>(p, i, v);
    else if (dt == kBF16) store_from_f32<kBF16>(p, i, v);
    else store_from_f32<kF16>(p, i, v);
}

}  // namespace coat
