// The clipped policy loss with a KL term over rows of logits x, and the gradient of the logits.
//
// For a row with token t:   logp = x[t] - lse,  lse = log sum exp x,  ratio = exp(logp - old),
//   loss  = -min(ratio A, clip(ratio, 1 - low, 1 + high) A) + kl (exp(ref - logp) - (ref - logp) - 1),
// averaged over the rows with the mask as weights; rows whose mask is 0 are not read. d loss / d logp is the row's `weight` (the free side of
// the minimum where the two are equal), and the logits' gradient weight * (1[v = t] - exp(x - lse)).
//
// Bound by memory: the forward pass reads the logits once, keeping a running maximum and the sum of exponentials below it; the
// backward pass reads them once and writes the gradient once. A token's own few values are computed in f64: next to the borders
// of the clipping the gradient jumps, and the logits are all that is large.
#include <algorithm>

#include "block_rows.hpp"

namespace hpt {

namespace {

// Exponentials are powers of two of x log2 e below a row's running maximum, which is kept in those units (any float near it serves). log2 e comes in two
// pieces: the float alone is 1e-8 of itself off, which would move every row's lse by 1e-8 of its distance below the maximum, all in one direction, and a loss that is the mean of
// terms of both signs shows that. The second piece is large against the first product's roundings (one next to the float's own last place would be rounded away every time).
// The sum's error is that of its terms weighted with their shares: each rounding of the argument costs a term |x - max| / 2^24, to either side.
constexpr double kLog2eExact = 1.4426950408889634;
constexpr float kLog2e = 1.4423828125f, kLog2eRest = (float)(kLog2eExact - 1.4423828125);  // (1477 / 1024, and what is left)
// The largest term's own argument is what rounding the maximum has left of it, and each argument is some 5e-12 of its logit off. That is harmless while the maximum is
// near: within kNear an argument is off by 2^-8 in every term alike, and by 5e-7 at most otherwise. From some 2e9 on it leaves the exponential's range, with infinities or zeros in place of 1.
// So no term is added while the maximum so far is beyond 2 kNear; if in the end it is within kNear, the terms left out were 0, and if it is not, the row is swept again by exact differences.
constexpr float kNear = 0x1p17f;

// (maximum in those units, sum of the powers below it) of two lanes or wavefronts.
__device__ __forceinline__ void meet(float& m, double& s, float m2, double s2) {
    const float n = fmaxf(m, m2);
    // (nothing seen is (-inf, 0); equal infinities are no distance apart; a NaN is in its sum)
    s = s * (double)(m == n ? 1.0f : __builtin_amdgcn_exp2f(m - n)) + s2 * (double)(m2 == n ? 1.0f : __builtin_amdgcn_exp2f(m2 - n));
    m = n;
}
__device__ __forceinline__ int64_t token_of(const void* token, int is64, int64_t row) {
    return is64 ? ((const int64_t*)token)[row] : (int64_t)((const int32_t*)token)[row];
}
__device__ __forceinline__ float mask_of(const PolicyArgs& a, int64_t row) {
    if (!a.mask) return 1.0f;
    return a.mask_bool ? (((const uint8_t*)a.mask)[row] ? 1.0f : 0.0f) : ((const float*)a.mask)[row];
}

// What a token brings along: read together, so that one latency covers all but the logit itself.
struct Token {
    int64_t id;
    float old, advantage, reference;
    __device__ __forceinline__ Token(const PolicyArgs& a, int64_t row) {
        id = token_of(a.token, a.token64, row);
        old = a.old_logp ? a.old_logp[row] : 0.0f;
        advantage = a.old_logp ? a.advantage[row] : 0.0f;
        reference = a.reference ? a.reference[row] : 0.0f;
    }
};
// The token's logit; NaN for a token outside the row.
template <class T> __device__ __forceinline__ float logit_of(const PolicyArgs& a, int64_t row, int64_t token) {
    return token >= 0 && token < a.cols ? Elem<T>::widen(((const T*)a.x + offset_of(a.kept, row))[token]) : __builtin_nanf("");
}

// What a row adds to the loss, and the loss's slope by its logp, both times the mask.
struct RowLoss {
    double loss, slope;
    __device__ __forceinline__ void store(const PolicyArgs& a, int64_t row) const {
        if (!a.old_logp) return;
        a.each[2 * row] = loss;
        a.each[2 * row + 1] = slope;  // (becomes the weight over the sum of the mask, in the last launch)
    }
};
// A row's results from its maximum, sum and token.
__device__ __forceinline__ RowLoss finish_row(const PolicyArgs& a, int64_t row, float mask, const Token& t, float xt, double m, double s) {
    const double rest = log(s), lse = m + rest;
    const double logp = ((double)xt - m) - rest;  // (exact differences first: m may be a type's lowest value)
    a.logp[row] = (float)logp;
    a.lse[row] = (float)lse;
    if (!a.old_logp) return {0.0, 0.0};
    const double adv = t.advantage, ratio = exp(logp - (double)t.old);
    const double low = 1.0 - a.clip_low, high = 1.0 + a.clip_high;
    const double free = ratio * adv, held = (ratio < low ? low : ratio > high ? high : ratio) * adv;
    double loss = free <= held ? -free : -held, slope = free <= held ? -free : 0.0;
    if (free != free || held != held) loss = slope = free + held;  // (a NaN is no side of the minimum)
    if (a.reference) {
        const double k = (double)t.reference - logp, e = exp(k);
        loss += a.kl_weight * (e - k - 1.0);
        slope += a.kl_weight * (1.0 - e);
    }
    return {loss * mask, slope * mask};
}
// A row that the mask leaves out.
__device__ __forceinline__ RowLoss skip_row(const PolicyArgs& a, int64_t row) {
    a.logp[row] = a.lse[row] = 0.0f;
    return {0.0, 0.0};
}

// Wavefronts on a SIMD: five as long as that needs no more than 96 registers (bf16 [8192, 50257] 167 us, with four of them, or with five and two registers spilled, 185); f16 needs a few more.
template <class T> constexpr int kStatsWaves = std::is_same<T, f16_t>::value ? 4 : 5;

// Maximum and sum of a part of a row. Vectors are aligned from the part's first aligned element on; the elements before it and behind the
// last whole vector are taken one by one. Four vectors of a thread are in flight together. Bound by memory: bf16 [8192, 50257] 153 us, 5.4 TB/s.
template <class T>
__global__ __launch_bounds__(256, kStatsWaves<T>) void policy_stats_kernel(const PolicyArgs a) {
    constexpr int VEC = 16 / sizeof(T), B = 4;
    __shared__ float most[4];
    __shared__ double sums[4];
    const float inf = __builtin_huge_valf();
    for (int64_t at = blockIdx.x; at < a.rows * a.split; at += gridDim.x) {
        const int64_t row = quotient(at, a.split);
        const int part = (int)(at - row * a.split);
        const float mask = mask_of(a, row);
        if (mask == 0.0f) {
            if (threadIdx.x == 0 && a.split == 1) skip_row(a, row).store(a, row);
            continue;  // (the same for the whole workgroup)
        }
        const int each = ((a.cols + a.split - 1) / a.split + VEC - 1) / VEC * VEC;
        const int e0 = min(part * each, a.cols), n = min(each, a.cols - e0);
        const T* x = (const T*)a.x + offset_of(a.kept, row) + e0;
        const int head = min(n, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T));
        const int vecs = (n - head) / VEC, tail = head + vecs * VEC;
        const T* body = x + head;
        float m = -inf;
        double s = 0.0;  // (as few as a thousand sums of 32 terms, one after the other in f32, would show in lse)
        auto take = [&](auto& v) {
            constexpr int N = sizeof(v) / sizeof(float);
            float t = v[0];
#pragma unroll
            for (int i = 1; i < N; ++i) t = fmaxf(t, v[i]);
            const float top = fmaxf(m, t * (float)kLog2eExact);
            float add = 0.0f;
            if (fabsf(top) < 2 * kNear) {
#pragma unroll
                for (int i = 0; i < N; ++i) add += __builtin_amdgcn_exp2f(fmaf(v[i], kLog2eRest, fmaf(v[i], kLog2e, -top)));
                s = s * (double)__builtin_amdgcn_exp2f(m - top) + (double)add;
                m = top;
            } else {  // nothing but masked logits yet, or logits far from zero: if that stays, the row is swept again below; what counts now is a NaN
#pragma unroll
                for (int i = 0; i < N; ++i) add += v[i] == v[i] ? 0.0f : v[i];
                s += (double)add;
                m = top;
            }
        };
        // (fewer than two vectors of single elements: a lane each)
        if ((int)threadIdx.x < head) {
            float v[1] = {Elem<T>::widen(x[threadIdx.x])};
            take(v);
        }
        if ((int)threadIdx.x < n - tail) {
            float v[1] = {Elem<T>::widen(x[tail + threadIdx.x])};
            take(v);
        }
        for (int v = threadIdx.x; v < vecs; v += B * 256) {
            Pack<T, VEC> p[B];
#pragma unroll
            for (int b = 0; b < B; ++b) {
                if (v + b * 256 < vecs) p[b] = load_pack<T, VEC>(body + (int64_t)(v + b * 256) * VEC);
                else
#pragma unroll
                    for (int i = 0; i < VEC; ++i) p[b].v[i] = Elem<T>::narrow(-inf);
            }
            float f[B * VEC];
#pragma unroll
            for (int b = 0; b < B; ++b)
#pragma unroll
                for (int i = 0; i < VEC; ++i) f[b * VEC + i] = Elem<T>::widen(p[b].v[i]);
            take(f);
        }
#pragma unroll
        for (int w = 1; w < 64; w <<= 1) meet(m, s, __shfl_xor(m, w, 64), shfl_xor_any(s, w));
        __syncthreads();
        if ((threadIdx.x & 63) == 0) {
            most[threadIdx.x >> 6] = m;
            sums[threadIdx.x >> 6] = s;
        }
        __syncthreads();
        m = most[0];
        s = sums[0];
        for (int w = 1; w < 4; ++w) meet(m, s, most[w], sums[w]);
        double top = (double)m / kLog2eExact;
        if (!(fabsf(m) < kNear) && n > 0) {
            // infinities, or finite logits far from zero (a row masked as a whole, or a part of one): element by element, by their differences from the largest
            // (loss alone, bf16 [8, 152000] with three quarters masked by -1e9, whole parts of the split rows among them, 15.8 us, without a mask 11.2).
            float t = -inf;
            for (int i = threadIdx.x; i < n; i += 256) t = fmaxf(t, Elem<T>::widen(x[i]));
            t = block_reduce<MaxF>(t, most);
            double add = 0.0;
            for (int i = threadIdx.x; i < n; i += 256) {
                const float v = Elem<T>::widen(x[i]);
                add += (double)(v == t ? 1.0f : __expf(v - t));
            }
            top = t;
            s = block_reduce<SumD>(add, sums);
        }
        if (threadIdx.x == 0) {
            if (a.split == 1) {
                const Token t(a, row);
                finish_row(a, row, mask, t, logit_of<T>(a, row, t.id), top, s).store(a, row);
            } else {
                a.partial[2 * at] = top;
                a.partial[2 * at + 1] = s;
            }
        }
    }
}

// A split row from its parts. They are weighted by the hardware's exponential, of f32 logits too: one of -D is off by D / 2^24 of itself or so, which is D e^-D / 2^24 of the row's sum at
// most, less than a rounding. The mask and what its token brings along are on their way together; a hidden row's logits are not read.
template <class T> __device__ __forceinline__ RowLoss join_row(const PolicyArgs& a, int64_t row, float mask) {
    const Token t(a, row);
    if (mask == 0.0f) return skip_row(a, row);
    const float xt = logit_of<T>(a, row, t.id);
    const double* p = a.partial + 2 * row * a.split;
    double m = -__builtin_huge_val(), s = 0.0;
    for (int k = 0; k < a.split; k += 8) {  // (eight parts on their way together)
        double most[8], sum[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int part = min(k + i, a.split - 1);
            most[i] = p[2 * part];
            sum[i] = p[2 * part + 1];
        }
        double n = m;
#pragma unroll
        for (int i = 0; i < 8; ++i) n = fmax(n, most[i]);
        // (equal infinities are no distance apart; a part of nothing is (-inf, 0))
        s *= (double)(m == n ? 1.0f : __expf((float)(m - n)));
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (k + i < a.split) s += sum[i] * (double)(most[i] == n ? 1.0f : __expf((float)(most[i] - n)));
        m = n;
    }
    return finish_row(a, row, mask, t, xt, m, s);
}
template <class T>
__global__ __launch_bounds__(64) void policy_rows_kernel(const PolicyArgs a) {
    const int64_t row = (int64_t)blockIdx.x * 64 + threadIdx.x;
    if (row < a.rows) join_row<T>(a, row, mask_of(a, row));
}

// The sums over the rows, in one workgroup and a fixed order: loss = sum of the losses / sum of the mask, and the weights over
// the same. Without a row that counts both are 0. Split rows (fewer than 2048) are joined on the way and stay with their thread
// (loss and gradient, f32 [1500, 32000] 107 -> 105 us, [64, 152000] 33 -> 31). f32 [640, 50257] 8 us, behind 25 and before 37 of the other two.
constexpr int kMostSplit = 2047;  // rows
template <class T>
__global__ __launch_bounds__(1024) void policy_sum_kernel(const PolicyArgs a) {
    __shared__ double place[2 * 16];
    double v[2] = {0.0, 0.0};
    double slope[2] = {0.0, 0.0};
    if (a.split > 1) {
        static_assert(kMostSplit <= 2 * 1024, "two rows a thread");
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int64_t row = threadIdx.x + k * 1024;
            if (row < a.rows) {
                const float mask = mask_of(a, row);
                const RowLoss l = join_row<T>(a, row, mask);
                v[0] += l.loss;
                v[1] += mask;
                slope[k] = l.slope;
            }
        }
    } else {
#pragma unroll 4
        for (int64_t row = threadIdx.x; row < a.rows; row += 1024) {
            v[0] += a.each[2 * row];
            v[1] += mask_of(a, row);
        }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int w = 1; w < 64; w <<= 1) v[k] += shfl_xor_any(v[k], w);
        if ((threadIdx.x & 63) == 0) place[2 * (threadIdx.x >> 6) + k] = v[k];
    }
    __syncthreads();
    double loss = 0.0, count = 0.0;
    for (int w = 0; w < 16; ++w) {
        loss += place[2 * w];
        count += place[2 * w + 1];
    }
    const double inv = count == 0.0 ? 0.0 : 1.0 / count;
    if (threadIdx.x == 0) a.loss[0] = (float)(loss * inv);
    if (a.split > 1) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int64_t row = threadIdx.x + k * 1024;
            if (row < a.rows) a.weight[row] = (float)(slope[k] * inv);
        }
    } else {
#pragma unroll 4
        for (int64_t row = threadIdx.x; row < a.rows; row += 1024) a.weight[row] = (float)(a.each[2 * row + 1] * inv);
    }
}

// The logits' gradient, piece by piece: no sums are left. A row of weight 0 is not read and has zeros, also where the loss's gradient is no finite number. Results leave as aligned vectors, logits come as
// they lie (aligned too where both start alike). bf16 [8192, 50257] 273 us, 6.0 TB/s of a read and a write.
template <class T>
__global__ __launch_bounds__(256) void policy_grad_kernel(const PolicyGradArgs a, int pieces, int each) {
    constexpr int VEC = 16 / sizeof(T);
    for (int64_t at = blockIdx.x; at < a.rows * pieces; at += gridDim.x) {
        const int64_t row = quotient(at, pieces);
        const int e0 = (int)(at - row * pieces) * each, n = min(each, a.cols - e0);
        T* out = (T*)a.out + row * a.cols + e0;
        const T* x = (const T*)a.x + offset_of(a.kept, row) + e0;
        const float weight = a.weight[row], w = weight == 0.0f ? 0.0f : weight * a.upstream, lse = a.lse[row];
        const int64_t t = token_of(a.token, a.token64, row) - e0;
        const int token = t >= 0 && t < n ? (int)t : -1;
        const int head = min(n, (int)((16 - ((uintptr_t)out & 15)) & 15) / (int)sizeof(T));
        const int vecs = (n - head) / VEC, tail = head + vecs * VEC;
        auto grad = [&](T v, int e) { return Elem<T>::narrow(w == 0.0f ? 0.0f : w * ((e == token ? 1.0f : 0.0f) - exp_row<T>(Elem<T>::widen(v) - lse))); };
        if ((int)threadIdx.x < head) out[threadIdx.x] = grad(w == 0.0f ? T{} : x[threadIdx.x], threadIdx.x);
        if ((int)threadIdx.x < n - tail) out[tail + threadIdx.x] = grad(w == 0.0f ? T{} : x[tail + threadIdx.x], tail + threadIdx.x);
        for (int v = threadIdx.x; v < vecs; v += 256) {
            const int e = head + v * VEC;
            Pack<T, VEC> p;
            __builtin_memset(&p, 0, sizeof p);
            if (w != 0.0f) p = load_pack_unaligned<T, VEC>(x + e);
#pragma unroll
            for (int i = 0; i < VEC; ++i) p.v[i] = grad(p.v[i], e + i);
            store_pack_stream<T, VEC>(out + e, p);
        }
    }
}

}  // namespace

int policy_split(int dtype, int64_t rows, int64_t cols) {
    if (rows == 0 || rows > kMostSplit) return 1;
    const int64_t bytes = cols * (int64_t)dtype_size(dtype);
    return (int)std::max<int64_t>(1, std::min<int64_t>({64, 4096 / rows, bytes / (16 << 10)}));
}

void launch_policy_loss(int dtype, const PolicyArgs& a, hipStream_t st) {
    HPT_WITH_TYPE(dtype, {
        if (a.rows > 0) policy_stats_kernel<T><<<(unsigned)std::min<int64_t>(a.rows * a.split, 1 << 20), 256, 0, st>>>(a);
        if (a.old_logp) policy_sum_kernel<T><<<1, 1024, 0, st>>>(a);
        else if (a.split > 1) policy_rows_kernel<T><<<(unsigned)((a.rows + 63) / 64), 64, 0, st>>>(a);
    });
}

void launch_policy_loss_backward(int dtype, const PolicyGradArgs& a, hipStream_t st) {
    HPT_WITH_TYPE(dtype, {
        constexpr int VEC = 16 / sizeof(T);
        // pieces of two vectors per thread, or nearly: us for one, two, four and eight, bf16 [8192, 50257] 328, 271, 275, 295, f32 [4096, 32000] 172, 157,
        // 165, 183 (fewer workgroups that walk the pieces: 390)
        const int most = 256 * 2 * VEC;
        const int pieces = (a.cols + most - 1) / most;
        const int each = ((a.cols + pieces - 1) / pieces + VEC - 1) / VEC * VEC;
        policy_grad_kernel<T><<<(unsigned)std::min<int64_t>(a.rows * pieces, 1 << 20), 256, 0, st>>>(a, pieces, each);
    });
}

}  // namespace hpt
