// Device-side pieces that the operators around a transformer's blocks share: a row's vectors in registers, whatever its length and
// alignment, and sums and maxima over the threads that hold it.
#pragma once

#include "block_entry.hpp"
#include "device_utils.hpp"

namespace hpt {

// a / b of numbers that are not negative: in 32 bits where both fit (a 64-bit division is some hundred instructions, and small launches wait
// for several of them before their first load).
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    if (((uint64_t)(a | b) >> 32) == 0) return (uint32_t)a / (uint32_t)b;
    return a / b;
}

struct SumF {
    __device__ static __forceinline__ float comb(float a, float b) { return a + b; }
};
// (Rows that are swept: a thread adds a vector's terms in f32 and the vectors in f64. One after the other in f32, the 2^19 of a row's longest share were up to 5e-3 off.)
struct SumD {
    __device__ static __forceinline__ double comb(double a, double b) { return a + b; }
};
struct MaxF {
    __device__ static __forceinline__ float comb(float a, float b) { return fmaxf(a, b); }
};
// The largest magnitude by its bits: they order as the magnitudes do, a NaN above everything.
struct MaxBits {
    __device__ static __forceinline__ uint32_t comb(uint32_t a, uint32_t b) { return a > b ? a : b; }
};

// Where vector v of a row of `cols` elements lies: it is taken from element `s` on, and its own elements are those from place `lo` on
// (VEC: none). AL: rows are whole, aligned vectors. Otherwise rows start anywhere (global memory takes unaligned vectors) and their last
// vector is taken from the row's end backwards, so that it reaches into the one before: rows of fewer elements than a vector holds have none.
template <int VEC, bool AL> struct Slot {
    int s, lo;
    __device__ __forceinline__ Slot(int v, int cols) {
        const int e = v * VEC;
        s = AL ? e : min(e, cols - VEC);
        lo = AL ? (e < cols ? 0 : VEC) : min(e - s, VEC);
    }
};

// The slot's vector, with what it holds of the one before; zeros where it has no element.
template <class T, bool AL> __device__ __forceinline__ Pack<T, 16 / sizeof(T)> load_slot(const T* row, const Slot<16 / sizeof(T), AL>& at) {
    constexpr int VEC = 16 / sizeof(T);
    Pack<T, VEC> p;
    if (at.lo < VEC) {
        if constexpr (AL) p = load_pack<T, VEC>(row + at.s);
        else p = load_pack_unaligned<T, VEC>(row + at.s);
    } else {
        __builtin_memset(&p, 0, sizeof p);
    }
    return p;
}
// Zeros in the places that are the vector's before. (Apart from the load, behind all of a row's: next to it, each load would be waited for before the next one
// is made: softmax with a bias f16 [1, 32, 1, 4097] 7.5 -> 7.0 us, norm f32 [3000, 7001] 33 -> 28.)
template <class T, bool AL> __device__ __forceinline__ void clean_slot(Pack<T, 16 / sizeof(T)>& p, const Slot<16 / sizeof(T), AL>& at) {
    constexpr int VEC = 16 / sizeof(T);
    if constexpr (!AL) {
        if (__any(at.lo & (VEC - 1))) {
            T zero;
            __builtin_memset(&zero, 0, sizeof zero);
#pragma unroll
            for (int i = 0; i < VEC; ++i) p.v[i] = i < at.lo ? zero : p.v[i];
        }
    }
}

// Only the slot's own elements are written: those before belong to another thread, which may not have read them yet where the result
// takes its operand's place. Whole vectors leave past the caches, which are left to the operands: norm bf16 [8192, 4096] in 8 bits with the sum
// 51.4 -> 48.7 us, softmax with a bias bf16 [8, 16, 1024, 1024] 102 -> 98; loads past the caches too gained nothing or lost (f16
// [13107, 5120] 90.3 -> 92.2).
template <class T, int VEC, bool AL> __device__ __forceinline__ void store_slot(T* row, const Slot<VEC, AL>& at, const Pack<T, VEC>& p) {
    if (at.lo == 0) {
        if constexpr (AL) store_pack_stream<T, VEC>(row + at.s, p);
        else if constexpr (sizeof(T) > 1) store_pack_unaligned_stream<T, VEC>(row + at.s, p);
        else store_pack_unaligned<T, VEC>(row + at.s, p);
    } else if constexpr (!AL) {
#pragma unroll
        for (int i = 1; i < VEC; ++i)
            if (i >= at.lo) row[at.s + i] = p.v[i];
    }
}

// Vector v of a row of any length, by elements at its end, zeros behind it: for the sweeps over rows that registers do not hold.
template <class T> __device__ __forceinline__ Pack<T, 16 / sizeof(T)> sweep_vec(const T* row, int v, int cols) {
    constexpr int VEC = 16 / sizeof(T);
    const int e = v * VEC;
    if (e + VEC <= cols) return load_pack_unaligned<T, VEC>(row + e);
    Pack<T, VEC> p;
    __builtin_memset(&p, 0, sizeof p);
    for (int i = 0; i < VEC && e + i < cols; ++i) p.v[i] = row[e + i];
    return p;
}
template <class T, int VEC> __device__ __forceinline__ void store_sweep_vec(T* row, int v, int cols, const Pack<T, VEC>& p) {
    const int e = v * VEC;
    if (e + VEC <= cols) store_pack_unaligned<T, VEC>(row + e, p);
    else
        for (int i = 0; i < VEC && e + i < cols; ++i) row[e + i] = p.v[i];
}

// N values at once folded over the threads of a row: the `tpr` lanes of a wavefront, or the whole workgroup (tpr > 64), whose
// wavefronts meet in LDS. `turn` alternates between two places of `smem` (2 * 16 * N values), so that one barrier is enough: nobody
// writes a place again before everybody has passed the barrier of the fold in between.
template <class Op, int N, class A> __device__ __forceinline__ void fold_row(A (&v)[N], int tpr, A* smem, int& turn) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = group_reduce<Op>(v[k], tpr < 64 ? tpr : 64);
    if (tpr > 64) {
        A* place = smem + turn * 16 * N;
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int k = 0; k < N; ++k) place[(threadIdx.x >> 6) * N + k] = v[k];
        }
        __syncthreads();
        const int waves = tpr >> 6;
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = place[k];
        for (int w = 1; w < waves; ++w) {
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] = Op::comb(v[k], place[w * N + k]);
        }
    }
}

// e^x: results of two bytes take the hardware's exponential, f32 ones the reduced form (x <= 0 up to a rounding).
template <class T> __device__ __forceinline__ float exp_row(float x) {
    if constexpr (sizeof(T) == 2) return __expf(x);
    else return exp_reduced<true>(x);
}

// The kernel of the wanted number of vectors per thread, or the next larger one that there is: up to 4 of two-byte types, up to 8 of f32
// (32 elements either way). Within HPT_WITH_TYPE.
#define HPT_WITH_NC(nc, ...)                                                            \
    do {                                                                                \
        constexpr bool kWide_ = sizeof(T) == 4;                                         \
        if ((nc) <= 1) { constexpr int NC = 1; __VA_ARGS__; }                           \
        else if ((nc) == 2) { constexpr int NC = 2; __VA_ARGS__; }                      \
        else if ((nc) == 3) { constexpr int NC = 3; __VA_ARGS__; }                      \
        else if ((nc) == 4 || !kWide_) { constexpr int NC = 4; __VA_ARGS__; }           \
        else if ((nc) <= 6) { constexpr int NC = kWide_ ? 6 : 4; __VA_ARGS__; }         \
        else { constexpr int NC = kWide_ ? 8 : 4; __VA_ARGS__; }                        \
    } while (0)
inline int most_vecs(int dtype) { return dtype == HPT_F32 ? 8 : 4; }

#define HPT_WITH_TYPE(dtype, ...)                                             \
    do {                                                                      \
        if ((dtype) == HPT_F16) { using T = f16_t; __VA_ARGS__; }             \
        else if ((dtype) == HPT_BF16) { using T = bf16_t; __VA_ARGS__; }      \
        else { using T = float; __VA_ARGS__; }                                \
    } while (0)

}  // namespace hpt
