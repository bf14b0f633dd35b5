// The divergence of a student's distribution over rows of logits x from a teacher's of which k entries (index, logit t) are known, at a temperature, and the
// gradient of the student's logits.
//
// With p = softmax(x / temperature) and q the teacher's probabilities of its entries, q = softmax(t / temperature) over them, or exp(t / temperature -
// teacher_lse) where the teacher's own log of the sum is given, in which case all other tokens count as one with r = max(0, 1 - sum q) against the student's s = 1 - sum p:
//   kl = sum q (log q - log p) + r (log r - log s),   loss = temperature^2 * the mean of kl over the rows, with the mask as weights.
// By x / temperature, a token's derivative is mass p - q (mass = sum q + r; q summed over entries that name it), and that of one which no entry names (mass - r / s) p.
//
// Bound by memory, as the policy loss is: one read forward, one read and one write backward. The entries (some hundred a row) come through LDS: as a bit for each token
// forward, where s is summed without the named tokens (1 - sum p would lose what is small), as a number for each token of a piece backward.
#include <algorithm>

#include "block_rows.hpp"

namespace hpt {

namespace {

constexpr double kLog2eD = 1.4426950408889634;
constexpr int kThreads = 256;
constexpr int kOwn = kMostEntries / kThreads;  // entries of a thread
constexpr int kBlock = 1 << 16;                // tokens that have a bit at a time

__device__ __forceinline__ float mask_of(const void* mask, int is_bool, int64_t row) {
    if (!mask) return 1.0f;
    return is_bool ? (((const uint8_t*)mask)[row] ? 1.0f : 0.0f) : ((const float*)mask)[row];
}
// An entry's token: -1 for none, `cols` for one outside the vocabulary.
__device__ __forceinline__ int token_of(const void* index, int is64, int64_t at, int cols) {
    const int64_t i = is64 ? ((const int64_t*)index)[at] : (int64_t)((const int32_t*)index)[at];
    return i < 0 ? -1 : i >= cols ? cols : (int)i;
}
__device__ __forceinline__ float logit_of(const void* t, int dtype, int64_t at) {
    if (dtype == HPT_F32) return ((const float*)t)[at];
    return dtype == HPT_F16 ? Elem<f16_t>::widen(((const f16_t*)t)[at]) : Elem<bf16_t>::widen(((const bf16_t*)t)[at]);
}

// (largest logit, sum of exponentials below it) of two lanes or wavefronts; `steps` = log2 e / temperature.
__device__ __forceinline__ void meet(float& m, double& s, float m2, double s2, float steps) {
    const float n = fmaxf(m, m2);
    // (nothing seen is (-inf, 0); equal infinities are no distance apart; a NaN is in its sum)
    s = s * (double)(m == n ? 1.0f : __builtin_amdgcn_exp2f((m - n) * steps)) + s2 * (double)(m2 == n ? 1.0f : __builtin_amdgcn_exp2f((m2 - n) * steps));
    m = n;
}

// What a row's parts have of it together.
struct RowSums {
    double most, sum;          // of the logits (of those that no entry names, where the rest counts)
    double named_most, named;  // of the others
    double teacher_most, a, b; // of the entries: sum e, sum e (t - x) / temperature with e = exp((t - teacher_most) / temperature)
};

// A row's divergence, and what its gradient needs: log2 of the sums that probabilities are over, in two pieces each (f32 alone would cost a gradient |lse| / 2^24 of itself).
__device__ __forceinline__ double finish_row(const DistillArgs& a, int64_t row, const RowSums& s) {
    const double inv = 1.0 / a.temperature, inf = __builtin_huge_val();
    auto scaled = [&](double x, double most) { return x == most ? 1.0 : exp((x - most) * inv); };
    double lse, rest = 0.0, kl, mass = 1.0, coef = 1.0, teacher;
    bool counts = true;
    if (!a.teacher_lse) {
        lse = rest = s.most * inv + log(s.sum);
        teacher = s.teacher_most * inv + log(s.a);
        kl = s.b / s.a - teacher + lse;
        counts = s.a != 0.0;
        if (!counts) kl = 0.0;
    } else {
        const double top = fmax(s.most, s.named_most);
        lse = top * inv + log(s.sum * scaled(s.most, top) + s.named * scaled(s.named_most, top));
        teacher = a.teacher_lse[row];
        const double part = s.a == 0.0 ? 0.0 : exp(s.teacher_most * inv - teacher), q = s.a * part;
        const bool others = s.sum != 0.0;
        double r = 1.0 - q;
        r = !others || r < 0.0 ? 0.0 : r;
        rest = others ? s.most * inv + log(s.sum) : lse;
        kl = (part == 0.0 ? 0.0 : part * s.b) + q * (lse - teacher) + (r == 0.0 ? 0.0 : r * (log(r) - (rest - lse)));
        if (q == 0.0) kl = r == 0.0 ? 0.0 : r * (log(r) - (rest - lse));
        mass = q + r;
        coef = others ? mass * exp(rest - lse) - r : 0.0;
    }
    a.kl[row] = (float)kl;
    float* t = a.terms + row * kTerms;
    auto pieces = [&](float* to, double v) {
        const float hi = (float)v;
        to[0] = hi;
        to[1] = fabsf(hi) < (float)inf ? (float)(v - (double)hi) : 0.0f;
    };
    pieces(t, lse * kLog2eD - log2(mass));
    pieces(t + 2, rest * kLog2eD);
    pieces(t + 4, teacher * kLog2eD);
    t[6] = (float)coef;
    t[7] = counts ? 1.0f : 0.0f;  // (becomes the weight in the last launch)
    return kl;
}
__device__ __forceinline__ void skip_row(const DistillArgs& a, int64_t row) {
    a.kl[row] = 0.0f;
    for (int i = 0; i < kTerms; ++i) a.terms[row * kTerms + i] = 0.0f;
}

// A row, or a part of one.
template <class T, bool REST>
__global__ __launch_bounds__(kThreads) void distill_stats_kernel(const DistillArgs a) {
    constexpr int VEC = 16 / sizeof(T), B = 4;
    const float inf = __builtin_huge_valf();
    __shared__ uint32_t bits[REST ? kBlock / 32 : 1];
    __shared__ float most[4];
    __shared__ double sums[4], sums2[4];
    __shared__ int again;
    const float steps = a.steps.hi + a.steps.lo;
    const double inv = 1.0 / a.temperature;
    for (int64_t at = blockIdx.x; at < a.rows * a.split; at += gridDim.x) {
        const int64_t row = quotient(at, a.split);
        const int part = (int)(at - row * a.split);
        if (mask_of(a.mask, a.mask_bool, row) == 0.0f) {
            if (threadIdx.x == 0 && a.split == 1) {
                skip_row(a, row);
                a.partial[at * kDistillPart] = 0.0;
            }
            continue;  // (the same for the whole workgroup)
        }
        const int each = ((a.cols + a.split - 1) / a.split + VEC - 1) / VEC * VEC;
        const int e0 = min(part * each, a.cols), e1 = min(e0 + each, a.cols);
        const T* x = (const T*)a.x + offset_of(a.kept, row);
        // the entries, and the student's logits of those in this part
        int token[kOwn];
        float t[kOwn], xt[kOwn];
        bool fresh[kOwn];  // (the first that names its token)
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const int j = threadIdx.x + i * kThreads;
            token[i] = -1;
            t[i] = -inf;
            if (j < a.k) {
                token[i] = token_of(a.index, a.index64, row * a.k + j, a.cols);
                if (token[i] >= 0) t[i] = logit_of(a.teacher, a.teacher_dtype, row * a.k + j);
            }
        }
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            xt[i] = token[i] >= e0 && token[i] < e1 ? Elem<T>::widen(x[token[i]]) : 0.0f;
            fresh[i] = false;
        }
        float m = -inf;
        double s = 0.0;
        auto take = [&](auto& v) {
            constexpr int N = sizeof(v) / sizeof(float);
            float top = v[0];
#pragma unroll
            for (int i = 1; i < N; ++i) top = fmaxf(top, v[i]);
            top = fmaxf(m, top);
            const float from = top == -inf ? 0.0f : top;
            float add = 0.0f;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float d = v[i] - from;
                add += __builtin_amdgcn_exp2f(fmaf(d, a.steps.hi, d * a.steps.lo));
            }
            s = s * (double)__builtin_amdgcn_exp2f((m - from) * steps) + (double)add;
            m = top;
        };
        for (int b0 = e0; b0 < e1; b0 += REST ? kBlock : e1 - e0) {
            const int b1 = REST ? min(b0 + kBlock, e1) : e1;
            if constexpr (REST) {
                __syncthreads();
                if (threadIdx.x == 0) again = 0;
                for (int i = threadIdx.x; i < (b1 - b0 + 31) / 32; i += kThreads) bits[i] = 0;
                __syncthreads();
#pragma unroll
                for (int i = 0; i < kOwn; ++i)
                    if (token[i] >= b0 && token[i] < b1) {
                        const uint32_t bit = 1u << ((token[i] - b0) & 31);
                        fresh[i] = !(atomicOr(&bits[(token[i] - b0) >> 5], bit) & bit);
                        if (!fresh[i]) again = 1;
                    }
                __syncthreads();
                if (again) {  // an index twice: the entry that comes first
#pragma unroll
                    for (int i = 0; i < kOwn; ++i)
                        if (token[i] >= b0 && token[i] < b1) {
                            const int j = threadIdx.x + i * kThreads;
                            fresh[i] = true;
                            for (int l = 0; l < j && fresh[i]; ++l) fresh[i] = token_of(a.index, a.index64, row * a.k + l, a.cols) != token[i];
                        }
                }
            }
            const int vecs = (b1 - b0) / VEC, tail = b0 + vecs * VEC;
            if ((int)threadIdx.x < b1 - tail) {
                const int e = tail + threadIdx.x;
                float v[1] = {Elem<T>::widen(x[e])};
                if constexpr (REST)
                    if (bits[(e - b0) >> 5] >> ((e - b0) & 31) & 1) v[0] = -inf;
                take(v);
            }
            for (int v = threadIdx.x; v < vecs; v += B * kThreads) {
                Pack<T, VEC> p[B];
#pragma unroll
                for (int b = 0; b < B; ++b) {
                    if (v + b * kThreads < vecs) p[b] = load_pack_unaligned<T, VEC>(x + b0 + (int64_t)(v + b * kThreads) * VEC);
                    else
#pragma unroll
                        for (int i = 0; i < VEC; ++i) p[b].v[i] = Elem<T>::narrow(-inf);
                }
                float f[B * VEC];
#pragma unroll
                for (int b = 0; b < B; ++b)
#pragma unroll
                    for (int i = 0; i < VEC; ++i) f[b * VEC + i] = Elem<T>::widen(p[b].v[i]);
                if constexpr (REST) {
                    uint32_t named[B], any = 0;
#pragma unroll
                    for (int b = 0; b < B; ++b) {
                        const int e = min(v + b * kThreads, vecs - 1) * VEC;
                        named[b] = bits[e >> 5] >> (e & 31) & ((1u << VEC) - 1);
                        any |= named[b];
                    }
                    if (__any(any != 0))
#pragma unroll
                        for (int b = 0; b < B; ++b)
#pragma unroll
                            for (int i = 0; i < VEC; ++i) f[b * VEC + i] = named[b] >> i & 1 ? -inf : f[b * VEC + i];
                }
                take(f);
            }
        }
#pragma unroll
        for (int w = 1; w < 64; w <<= 1) meet(m, s, __shfl_xor(m, w, 64), shfl_xor_any(s, w), steps);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) {
            most[threadIdx.x >> 6] = m;
            sums[threadIdx.x >> 6] = s;
        }
        __syncthreads();
        m = most[0];
        s = sums[0];
        for (int w = 1; w < 4; ++w) meet(m, s, most[w], sums[w], steps);
        // the teacher's entries
        float teacher_most = -inf, named_most = -inf;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            teacher_most = fmaxf(teacher_most, t[i]);
            if (REST && fresh[i]) named_most = fmaxf(named_most, xt[i]);
            bad |= token[i] == a.cols;
        }
        teacher_most = block_reduce<MaxF>(teacher_most, most);
        if constexpr (REST) named_most = block_reduce<MaxF>(named_most, most);
        double ea = 0.0, eb = 0.0, named = 0.0;
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
            if (token[i] >= e0 && token[i] < e1) {
                const double e = t[i] == -inf ? 0.0 : exp(((double)t[i] - (double)teacher_most) * inv);
                ea += e;
                if (e != 0.0) eb += e * (((double)t[i] - (double)xt[i]) * inv);
                if (REST && fresh[i]) named += xt[i] == -inf ? 0.0 : exp(((double)xt[i] - (double)named_most) * inv);
            }
        if (bad && part == 0) ea = __builtin_nan("");
        ea = block_reduce<SumD>(ea, sums2);
        eb = block_reduce<SumD>(eb, sums);
        if constexpr (REST) named = block_reduce<SumD>(named, sums2);
        if (threadIdx.x == 0) {
            double* p = a.partial + at * kDistillPart;
            const RowSums r{m, s, named_most, named, teacher_most, ea, eb};
            if (a.split == 1) {
                p[0] = finish_row(a, row, r);
            } else {
                p[0] = r.most;
                p[1] = r.sum;
                p[2] = r.named_most;
                p[3] = r.named;
                p[4] = r.teacher_most;
                p[5] = r.a;
                p[6] = r.b;
            }
        }
    }
}

// A split row from its parts, a lane each.
__global__ __launch_bounds__(64) void distill_rows_kernel(const DistillArgs a) {
    const int64_t row = blockIdx.x;
    double* p = a.partial + row * a.split * kDistillPart;
    if (mask_of(a.mask, a.mask_bool, row) == 0.0f) {
        if (threadIdx.x == 0) {
            skip_row(a, row);
            p[0] = 0.0;
        }
        return;
    }
    const double inf = __builtin_huge_val(), inv = 1.0 / a.temperature;
    RowSums r{-inf, 0.0, -inf, 0.0, -inf, 0.0, 0.0};
    if ((int)threadIdx.x < a.split) {
        const double* q = p + threadIdx.x * kDistillPart;
        r = {q[0], q[1], q[2], q[3], q[4], q[5], q[6]};
    }
    auto meet = [&](double& m, double& s) {
#pragma unroll
        for (int w = 1; w < 64; w <<= 1) {
            const double m2 = shfl_xor_any(m, w), s2 = shfl_xor_any(s, w), n = fmax(m, m2);
            const double f1 = m == n ? 1.0 : exp((m - n) * inv), f2 = m2 == n ? 1.0 : exp((m2 - n) * inv);
            s = s * f1 + s2 * f2;
            m = n;
        }
    };
    meet(r.most, r.sum);
    if (a.teacher_lse) meet(r.named_most, r.named);
    r.a = group_reduce<SumD>(r.a, 64);
    r.b = group_reduce<SumD>(r.b, 64);
    if (threadIdx.x == 0) p[0] = finish_row(a, row, r);
}

// The sums over the rows, in one workgroup and a fixed order, and each row's weight. Without a row that counts all are 0.
__global__ __launch_bounds__(1024) void distill_sum_kernel(const DistillArgs a) {
    __shared__ double place[16];
    double loss = 0.0, count = 0.0;
#pragma unroll 4
    for (int64_t row = threadIdx.x; row < a.rows; row += 1024) {
        const float mask = mask_of(a.mask, a.mask_bool, row);
        if (mask != 0.0f) {
            loss += a.partial[row * a.split * kDistillPart] * mask;
            count += mask;
        }
    }
    loss = block_reduce<SumD>(loss, place);
    count = block_reduce<SumD>(count, place);
    const double inv = count == 0.0 ? 0.0 : 1.0 / count;
    if (threadIdx.x == 0) a.loss[0] = (float)(loss * inv * a.temperature * a.temperature);
#pragma unroll 4
    for (int64_t row = threadIdx.x; row < a.rows; row += 1024)
        a.terms[row * kTerms + 7] *= (float)(mask_of(a.mask, a.mask_bool, row) * inv * a.temperature);
}

// The logits' gradient, piece by piece. A row of weight 0 is not read and has zeros.
template <class T>
__global__ __launch_bounds__(kThreads) void distill_grad_kernel(const DistillGradArgs a, int pieces, int each) {
    constexpr int VEC = 16 / sizeof(T), N = 2;
    __shared__ float probs[kThreads * N * VEC];  // the teacher's of the piece's tokens, -1 where no entry names one
    __shared__ int again;
    for (int64_t at = blockIdx.x; at < a.rows * pieces; at += gridDim.x) {
        const int64_t row = quotient(at, pieces);
        const int e0 = (int)(at - row * pieces) * each, n = min(each, a.cols - e0);
        T* out = (T*)a.out + row * a.cols + e0;
        const T* x = (const T*)a.x + offset_of(a.kept, row) + e0;
        const float* terms = a.terms + row * kTerms;
        const float weight = terms[7], w = weight == 0.0f ? 0.0f : weight * a.upstream;
        const bool on = weight != 0.0f;
        // results leave as aligned vectors, logits come as they lie
        const int head = min(n, (int)((16 - ((uintptr_t)out & 15)) & 15) / (int)sizeof(T));
        const int vecs = (n - head) / VEC, tail = head + vecs * VEC;
        Pack<T, VEC> p[N];
        T first, last;
        __builtin_memset(p, 0, sizeof p);
        __builtin_memset(&first, 0, sizeof first);
        __builtin_memset(&last, 0, sizeof last);
        if (on) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int v = threadIdx.x + i * kThreads;
                if (v < vecs) p[i] = load_pack_unaligned<T, VEC>(x + head + v * VEC);
            }
            if ((int)threadIdx.x < head) first = x[threadIdx.x];
            if ((int)threadIdx.x < n - tail) last = x[tail + threadIdx.x];
        }
        const float base_hi = terms[0], base_lo = terms[1], rest_hi = terms[2], rest_lo = terms[3], coef = terms[6];
        const double teacher = (double)terms[4] + (double)terms[5];
        auto prob = [&](int j) { return (float)exp2((double)logit_of(a.teacher, a.teacher_dtype, row * a.k + j) * (kLog2eD / a.temperature) - teacher); };
        if (on) {
            __syncthreads();
            for (int i = threadIdx.x; i < n; i += kThreads) probs[i] = -1.0f;
            if (threadIdx.x == 0) again = 0;
            __syncthreads();
            for (int j = threadIdx.x; j < a.k; j += kThreads) {
                const int e = token_of(a.index, a.index64, row * a.k + j, a.cols) - e0;
                if (e >= 0 && e < n && e + e0 < a.cols) {
                    const uint32_t old = atomicExch((uint32_t*)&probs[e], __float_as_uint(prob(j)));
                    if (old != __float_as_uint(-1.0f)) again = 1;
                }
            }
            __syncthreads();
            if (again) {  // an index twice: the sum, in the entries' order
                for (int i = threadIdx.x; i < n; i += kThreads) probs[i] = -1.0f;
                __syncthreads();
                if (threadIdx.x == 0)
                    for (int j = 0; j < a.k; ++j) {
                        const int e = token_of(a.index, a.index64, row * a.k + j, a.cols) - e0;
                        if (e >= 0 && e < n && e + e0 < a.cols) probs[e] = (probs[e] == -1.0f ? 0.0f : probs[e]) + prob(j);
                    }
                __syncthreads();
            }
        }
        auto grad = [&](T v, int e) {
            if (!on) return Elem<T>::narrow(0.0f);
            const float q = probs[e], f = Elem<T>::widen(v);
            const bool named = !(q == -1.0f);
            const float y = __builtin_amdgcn_exp2f(fmaf(f, a.steps.hi, named ? -base_hi : -rest_hi) + fmaf(f, a.steps.lo, named ? -base_lo : -rest_lo));
            return Elem<T>::narrow(w * (named ? y - q : coef * y));
        };
        if ((int)threadIdx.x < head) out[threadIdx.x] = grad(first, threadIdx.x);
        if ((int)threadIdx.x < n - tail) out[tail + threadIdx.x] = grad(last, tail + threadIdx.x);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int v = threadIdx.x + i * kThreads;
            if (v >= vecs) continue;
            const int e = head + v * VEC;
#pragma unroll
            for (int l = 0; l < VEC; ++l) p[i].v[l] = grad(p[i].v[l], e + l);
            store_pack_stream<T, VEC>(out + e, p[i]);
        }
    }
}

}  // namespace

int distill_split(int dtype, int64_t rows, int64_t cols) {
    if (rows == 0 || rows > 2047) return 1;
    const int64_t bytes = cols * (int64_t)dtype_size(dtype);
    return (int)std::max<int64_t>(1, std::min<int64_t>({64, 4096 / rows, bytes / (16 << 10)}));
}

void launch_distill_loss(int dtype, const DistillArgs& a, hipStream_t st) {
    if (a.rows > 0) {
        HPT_WITH_TYPE(dtype, {
            const unsigned blocks = (unsigned)std::min<int64_t>(a.rows * a.split, 1 << 20);
            if (a.teacher_lse) distill_stats_kernel<T, true><<<blocks, kThreads, 0, st>>>(a);
            else distill_stats_kernel<T, false><<<blocks, kThreads, 0, st>>>(a);
        });
        if (a.split > 1) distill_rows_kernel<<<(unsigned)a.rows, 64, 0, st>>>(a);
    }
    distill_sum_kernel<<<1, 1024, 0, st>>>(a);
}

void launch_distill_loss_backward(int dtype, const DistillGradArgs& a, hipStream_t st) {
    HPT_WITH_TYPE(dtype, {
        constexpr int VEC = 16 / sizeof(T);
        const int most = kThreads * 2 * VEC;
        const int pieces = (a.cols + most - 1) / most;
        const int each = ((a.cols + pieces - 1) / pieces + VEC - 1) / VEC * VEC;
        distill_grad_kernel<T><<<(unsigned)std::min<int64_t>(a.rows * pieces, 1 << 20), kThreads, 0, st>>>(a, pieces, each);
    });
}

}  // namespace hpt
