// The divergence of a student's distribution over rows of logits x from a teacher's of which k entries (index, logit t) are known, at a temperature, and the
// gradient of the student's logits.
//
// With p = softmax(x / temperature) and q the teacher's probabilities of its entries, q = softmax(t / temperature) over them, or exp(t / temperature -
// teacher_lse) where the teacher's own log of the sum is given, in which case all other tokens count as one with r = max(0, 1 - sum q) against the student's s = 1 - sum p:
//   kl = sum q (log q - log p) + r (log r - log s),   loss = temperature^2 * the mean of kl over the rows, with the mask as weights.
// By x / temperature, a token's derivative is mass p - q (mass = sum q + r; q summed over entries that name it), and that of one which no entry names (mass - r / s) p.
// All of it from distances below the largest logit and the largest entry, so rows may lie anywhere.
//
// Bound by memory, as the policy loss is: one read forward, one read and one write backward. The entries (some hundred a row) come through LDS: as a bit for each token
// forward, where s is summed without the named tokens (1 - sum p would lose what is small), as a number for each token of a piece backward.
// bf16 [8192, 50257], k = 64, with the rest: 142 us forward (5.8 TB/s), 22 of the launch that joins the rows' parts with their entries, 4 of the mean over the rows, 289 backward (5.7 TB/s).
#include <algorithm>

#include "vocab_rows.hpp"

namespace hpt {

namespace {

constexpr double kLog2eD = 1.4426950408889634;
constexpr int kThreads = 256;
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

// The exponential of a distance over the temperature.
__device__ __forceinline__ float exp_of(float d, const Steps& steps) { return __builtin_amdgcn_exp2f(fmaf(d, steps.hi, d * steps.lo)); }

// (largest logit, sum of exponentials below it) of two lanes or wavefronts.
__device__ __forceinline__ void meet(float& m, double& s, float m2, double s2, const Steps& steps) {
    const float n = fmaxf(m, m2);
    // (nothing seen is (-inf, 0); equal infinities are no distance apart; a NaN is in its sum)
    s = s * (double)(m == n ? 1.0f : exp_of(m - n, steps)) + s2 * (double)(m2 == n ? 1.0f : exp_of(m2 - n, steps));
    m = n;
}

// Wavefronts on a SIMD.
template <class T> constexpr int kStatsWaves = 5;
constexpr int kGradVecs = 4;  // vectors of a lane

// What a row's parts have of it together.
struct RowSums {
    double most, sum;          // of the logits (of those that no entry names, where the rest counts)
    double named_most, named;  // of the others
    // of the entries: sum e, sum e ((t - teacher_most) - (x - the larger of most and named_most)) / temperature with e = exp((t - teacher_most) / temperature)
    double teacher_most, a, b;
};

// A row's divergence, and what its gradient needs. Logits count by their distances below the largest alone, the teacher's too (but for its own log of the sum): they may lie anywhere, as in a
// row of which a mask has left nothing but -1e9 or the type's lowest value. Terms: 0 the largest logit, 1 what a named token's exponential below it is multiplied by; 2 and 3 the same of an
// unnamed one; 4 and 5 the same of an entry's; 7 the weight.
__device__ __forceinline__ double finish_row(const DistillArgs& a, int64_t row, const RowSums& s) {
    const double inv = 1.0 / a.temperature;
    float* t = a.terms + row * kTerms;
    double kl;
    if (!a.teacher_lse) {
        kl = s.a == 0.0 ? 0.0 : s.b / s.a - log(s.a) + log(s.sum);
        t[0] = t[2] = (float)s.most;
        t[1] = t[3] = (float)(1.0 / s.sum);
        t[4] = (float)s.teacher_most;
        t[5] = (float)(1.0 / s.a);
    } else {
        // (one exponential for both sums' distance; equal infinities are no distance apart)
        const bool below = s.most < s.named_most;
        const double far = s.most == s.named_most ? 1.0 : exp(-fabs(s.most - s.named_most) * inv);
        const double left = s.sum * (below ? far : 1.0), all = left + s.named * (below ? 1.0 : far), log_all = log(all);
        const double largest = fmax(s.most, s.named_most), beyond = s.teacher_most * inv - a.teacher_lse[row];
        const double part = s.a == 0.0 ? 0.0 : exp(beyond), q = s.a * part;
        const bool others = s.sum != 0.0;
        double r = 1.0 - q, mass = 1.0;
        if (!others || r < 0.0) {
            r = 0.0;
            mass = q;
        }
        kl = r == 0.0 ? 0.0 : r * (log(r) - ((s.most - largest) * inv + log(s.sum) - log_all));
        if (q != 0.0) kl += part * s.b + q * (beyond + log_all);
        t[0] = (float)largest;
        t[1] = (float)(mass / all);
        t[2] = (float)(others ? s.most : largest);
        t[3] = others ? (float)((mass * (left / all) - r) / s.sum) : 0.0f;
        t[4] = s.a == 0.0 ? 0.0f : (float)s.teacher_most;
        t[5] = (float)part;
    }
    a.kl[row] = (float)kl;
    t[6] = 0.0f;
    t[7] = a.teacher_lse || s.a != 0.0 ? 1.0f : 0.0f;  // (becomes the weight in the last launch)
    return kl;
}
__device__ __forceinline__ void skip_row(const DistillArgs& a, int64_t row) {
    a.kl[row] = 0.0f;
    for (int i = 0; i < kTerms; ++i) a.terms[row * kTerms + i] = 0.0f;
}

// Largest logit and sum of exponentials of a row, or of a part of one; where the rest counts, of the tokens that no entry names (a bit each tells).
template <class T, bool REST>
__global__ __launch_bounds__(kThreads, kStatsWaves<T>) void distill_stats_kernel(const DistillArgs a) {
    constexpr int VEC = 16 / sizeof(T), B = 4;
    const float inf = __builtin_huge_valf();
    __shared__ uint32_t bits[REST ? kBlock / 32 + 1 : 1];
    __shared__ float most[4];
    __shared__ double sums[4];
    __shared__ int again;  // a token is named twice
    for (int64_t at = blockIdx.x; at < a.rows * a.split; at += gridDim.x) {
        const int64_t row = quotient(at, a.split);
        const int part = (int)(at - row * a.split);
        if (mask_of(a.mask, a.mask_bool, row) == 0.0f) continue;  // (the same for the whole workgroup)
        const int each = ((a.cols + a.split - 1) / a.split + VEC - 1) / VEC * VEC;
        const int e0 = min(part * each, a.cols), e1 = min(e0 + each, a.cols);
        const T* x = (const T*)a.x + offset_of(a.kept, row);
        if (threadIdx.x == 0) again = 0;  // (the thread that reads it)
        float m = -inf;
        double s = 0.0;
        auto take = [&](auto& v) {
            constexpr int N = sizeof(v) / sizeof(float);
            float top = v[0];
#pragma unroll
            for (int i = 1; i < N; ++i) top = fmaxf(top, v[i]);
            top = fmaxf(m, top);
            const float from = top == -inf ? 0.0f : top;
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = exp_of(v[i] - from, a.steps);
            s = s * (double)exp_of(m - from, a.steps) + (double)sum_by_twos(v);
            m = top;
        };
        for (int b0 = e0; b0 < e1; b0 += REST ? kBlock : e1 - e0) {
            const int b1 = REST ? min(b0 + kBlock, e1) : e1;
            // vectors are aligned from the block's first aligned logit on; a token's bit stands so that those of a vector stand together
            const int head = min(b1 - b0, (int)((16 - ((uintptr_t)(x + b0) & 15)) & 15) / (int)sizeof(T));
            const int vecs = (b1 - b0 - head) / VEC, tail = b0 + head + vecs * VEC, first = b0 + head - VEC;
            const T* body = x + b0 + head;
            auto named = [&](int e) { return bits[(e - first) >> 5] >> ((e - first) & 31); };
            if constexpr (REST) {
                __syncthreads();
                for (int i = threadIdx.x; i <= (b1 - first) / 32; i += kThreads) bits[i] = 0;
                __syncthreads();
                for (int j = threadIdx.x; j < a.k; j += kThreads) {
                    const int e = token_of(a.index, a.index64, row * a.k + j, a.cols);
                    if (e >= b0 && e < b1) {
                        const uint32_t bit = 1u << ((e - first) & 31);
                        if (atomicOr(&bits[(e - first) >> 5], bit) & bit) again = 1;
                    }
                }
                __syncthreads();
            }
            // (fewer than two vectors of single logits: a lane each)
            auto single = [&](int e) {
                float v[1] = {Elem<T>::widen(x[e])};
                if constexpr (REST)
                    if (named(e) & 1) v[0] = -inf;
                take(v);
            };
            if ((int)threadIdx.x < head) single(b0 + threadIdx.x);
            if ((int)threadIdx.x < b1 - tail) single(tail + threadIdx.x);
            // (no load hangs on a condition: the compiler would wait for each before the next)
            for (int v0 = 0; v0 < vecs; v0 += B * kThreads) {
                Pack<T, VEC> p[B];
#pragma unroll
                for (int b = 0; b < B; ++b) p[b] = load_pack_stream<T, VEC>(body + (int64_t)min(v0 + (int)threadIdx.x + b * kThreads, vecs - 1) * VEC);
                if constexpr (REST) {
                    uint32_t some[B], any = 0;
#pragma unroll
                    for (int b = 0; b < B; ++b) {
                        some[b] = named(b0 + head + min(v0 + (int)threadIdx.x + b * kThreads, vecs - 1) * VEC) & ((1u << VEC) - 1);
                        any |= some[b];
                    }
                    if (any != 0) {
#pragma unroll
                        for (int b = 0; b < B; ++b)
#pragma unroll
                            for (int i = 0; i < VEC; ++i)
                                if (some[b] >> i & 1) p[b].v[i] = Elem<T>::narrow(-inf);
                    }
                }
                if (v0 + B * kThreads > vecs) {
#pragma unroll
                    for (int b = 0; b < B; ++b)
                        if (v0 + (int)threadIdx.x + b * kThreads >= vecs)
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
        }
#pragma unroll
        for (int w = 1; w < 64; w <<= 1) meet(m, s, __shfl_xor(m, w, 64), shfl_xor_any(s, w), a.steps);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) {
            most[threadIdx.x >> 6] = m;
            sums[threadIdx.x >> 6] = s;
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            m = most[0];
            s = sums[0];
            for (int w = 1; w < 4; ++w) meet(m, s, most[w], sums[w], a.steps);
            double* p = a.partial + at * kDistillPart;
            p[0] = m;
            p[1] = s;
            p[2] = again ? 1.0 : 0.0;
        }
    }
}

// A row's sums from its parts (at most 64, a lane each) and its entries, for a wavefront.
template <class T> __device__ __forceinline__ RowSums sums_of_row(const DistillArgs& a, int64_t row) {
    const int lane = threadIdx.x & 63;
    const double inf = __builtin_huge_val(), inv = 1.0 / a.temperature;
    const T* x = (const T*)a.x + offset_of(a.kept, row);
    RowSums r{-inf, 0.0, -inf, 0.0, -inf, 0.0, 0.0};
    double twice = 0.0;
    if (lane < a.split) {
        const double* p = a.partial + (row * a.split + lane) * kDistillPart;
        r.most = p[0];
        r.sum = p[1];
        twice = p[2];
    }
    // the entries: four of a lane at a time on their way together
    struct Entry {
        int token;
        float t, x;
    };
    auto entry = [&](int j) {
        Entry e{-1, -(float)inf, 0.0f};
        if (j < a.k) {
            e.token = token_of(a.index, a.index64, row * a.k + j, a.cols);
            if (e.token >= 0) e.t = logit_of(a.teacher, a.teacher_dtype, row * a.k + j);
            if (e.token >= 0 && e.token < a.cols) e.x = Elem<T>::widen(x[e.token]);
        }
        return e;
    };
    float teacher_most = -(float)inf, named_most = -(float)inf;
    bool bad = false;
    const bool rest = a.teacher_lse != nullptr;
    Entry few[4];
    for (int j0 = 0; j0 < a.k; j0 += 256) {
#pragma unroll
        for (int i = 0; i < 4; ++i) few[i] = entry(j0 + i * 64 + lane);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            teacher_most = fmaxf(teacher_most, few[i].t);
            if (few[i].token >= 0) named_most = fmaxf(named_most, few[i].x);
            bad |= few[i].token == a.cols;
        }
    }
    teacher_most = group_reduce<MaxF>(teacher_most, 64);
    named_most = group_reduce<MaxF>(named_most, 64);
    // the parts together
    if (a.split > 1) {
        double most = r.most;
#pragma unroll
        for (int w = 1; w < 64; w <<= 1) most = fmax(most, shfl_xor_any(most, w));
        if (r.sum != 0.0) r.sum *= exp((r.most - most) * inv);
        r.sum = group_reduce<SumD>(r.sum, 64);
        r.most = most;
    } else {
        r.sum = lane_of(r.sum, 0);
        r.most = lane_of(r.most, 0);
    }
    const double largest = fmax(r.most, (double)named_most);
    for (int j0 = 0; j0 < a.k; j0 += 256) {
        if (a.k > 256)
#pragma unroll
            for (int i = 0; i < 4; ++i) few[i] = entry(j0 + i * 64 + lane);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const Entry& e = few[i];
            if (e.token < 0 || e.token == a.cols) continue;
            const double p = e.t == -(float)inf ? 0.0 : exp(((double)e.t - (double)teacher_most) * inv);
            r.a += p;
            if (p != 0.0) r.b += p * ((((double)e.t - (double)teacher_most) - ((double)e.x - largest)) * inv);
        }
        if (rest) {
            // the student's, each token once: where one is named twice, an entry whose token one before it names is passed over
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const Entry& e = few[i];
                bool first = e.token >= 0 && e.token < a.cols && e.x != -(float)inf;
                if (__any(twice != 0.0)) {
                    const int j = j0 + i * 64 + lane;
                    for (int l = 0; l < j && first; ++l) first = token_of(a.index, a.index64, row * a.k + l, a.cols) != e.token;
                }
                if (first) r.named += exp(((double)e.x - (double)named_most) * inv);
            }
        }
    }
    if (__any(bad)) r.a = __builtin_nan("");
    r.a = group_reduce<SumD>(r.a, 64);
    r.b = group_reduce<SumD>(r.b, 64);
    r.named = group_reduce<SumD>(r.named, 64);
    r.teacher_most = teacher_most;
    r.named_most = named_most;
    return r;
}

// Rows from their sums: a wavefront takes one, and those of a workgroup are finished together, a lane each (the logarithms and exponentials of 64 bits are some thousand
// instructions, for one lane as for all).
constexpr int kRowsAtOnce = 16;
template <class T>
__global__ __launch_bounds__(64 * kRowsAtOnce, 8) void distill_rows_kernel(const DistillArgs a, int64_t from) {
    __shared__ RowSums sums[kRowsAtOnce];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row0 = from + (int64_t)blockIdx.x * kRowsAtOnce;
    if (row0 + wave < a.rows && mask_of(a.mask, a.mask_bool, row0 + wave) != 0.0f) {
        const RowSums r = sums_of_row<T>(a, row0 + wave);
        if ((threadIdx.x & 63) == 0) sums[wave] = r;
    }
    __syncthreads();
    const int64_t row = row0 + threadIdx.x;
    if (threadIdx.x >= kRowsAtOnce || row >= a.rows) return;
    if (mask_of(a.mask, a.mask_bool, row) == 0.0f) {
        skip_row(a, row);
        a.each[row] = 0.0;
    } else {
        a.each[row] = finish_row(a, row, sums[threadIdx.x]);
    }
}

// The sums over the rows, in one workgroup and a fixed order, and each row's weight. Without a row that counts all are 0.
__global__ __launch_bounds__(1024) void distill_sum_kernel(const DistillArgs a) {
    __shared__ double place[2 * 16];
    double loss = 0.0, count = 0.0;
#pragma unroll 4
    for (int64_t row = threadIdx.x; row < a.rows; row += 1024) {
        const float mask = mask_of(a.mask, a.mask_bool, row);
        if (mask != 0.0f) {
            loss += a.each[row] * mask;
            count += mask;
        }
    }
    loss = group_reduce<SumD>(loss, 64);
    count = group_reduce<SumD>(count, 64);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (lane == 0) {
        place[wave] = loss;
        place[16 + wave] = count;
    }
    __syncthreads();
    // (every wavefront for itself, both sums side by side: one read of LDS)
    const double both = group_reduce<SumD>(place[lane & 31], 16);
    loss = lane_of(both, 0);
    count = lane_of(both, 16);
    const double inv = count == 0.0 ? 0.0 : 1.0 / count;
    if (threadIdx.x == 0) a.loss[0] = (float)(loss * inv * a.temperature * a.temperature);
#pragma unroll 4
    for (int64_t row = threadIdx.x; row < a.rows; row += 1024)
        a.terms[row * kTerms + 7] *= (float)(mask_of(a.mask, a.mask_bool, row) * inv * a.temperature);
}

// The logits' gradient, a piece for each wavefront, which waits for nobody. A row of weight 0 is not read and has zeros. Every lane has what its tokens' vectors get if no
// entry names them; a named token (a bit tells) is left out there and written by the lane of the first entry that names it.
template <class T>
__global__ __launch_bounds__(kThreads) void distill_grad_kernel(const DistillGradArgs a, int pieces, int each) {
    constexpr int VEC = 16 / sizeof(T), N = kGradVecs, WORDS = (64 * N * VEC + VEC + 31) / 32;
    __shared__ uint32_t shared_bits[kThreads / 64][WORDS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t* bits = shared_bits[wave];
    auto fence = [] { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); };  // (a wavefront's accesses to LDS are in order)
    for (int64_t at = (int64_t)blockIdx.x * (kThreads / 64) + wave; at < a.rows * pieces; at += (int64_t)gridDim.x * (kThreads / 64)) {
        const int64_t row = quotient(at, pieces);
        const int e0 = (int)(at - row * pieces) * each, n = min(each, a.cols - e0);
        T* out = (T*)a.out + row * a.cols + e0;
        const T* x = (const T*)a.x + offset_of(a.kept, row) + e0;
        const float* terms = a.terms + row * kTerms;
        const float weight = terms[7], w = weight == 0.0f ? 0.0f : weight * a.upstream;
        const bool on = weight != 0.0f;
        auto token = [&](int j) { return token_of(a.index, a.index64, row * a.k + j, a.cols); };
        int named = lane < a.k ? token(lane) : -1;
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
            for (int i = 0; i < N; ++i)
                if (lane + i * 64 < vecs) p[i] = load_pack_unaligned<T, VEC>(x + head + (lane + i * 64) * VEC);
            if (lane < head) first = x[lane];
            if (lane < n - tail) last = x[tail + lane];
        }
        const float rest_most = terms[2], coef = w * terms[3];
        // a token's bit stands so that those of a vector stand together
        const int shift = VEC - head;
        if (on) {
            for (int i = lane; i < WORDS; i += 64) bits[i] = 0;
            fence();
            uint32_t mine = 0;  // entries of this lane that name a token of the piece
            bool twice = false;
            for (int i = 0; i * 64 < a.k; ++i) {
                if (i) named = i * 64 + lane < a.k ? token(i * 64 + lane) : -1;
                const int e = named - e0;
                if (e >= 0 && e < n) {
                    const int b = e + shift;
                    twice |= atomicOr(&bits[b >> 5], 1u << (b & 31)) >> (b & 31) & 1;
                    mine |= 1u << i;
                }
            }
            static_assert(kMostEntries <= 64 * 32, "a bit for each entry of a lane");
            twice = __any(twice);
            fence();
            while (mine) {
                const int j = __builtin_ctz(mine) * 64 + lane, e = token(j);
                mine &= mine - 1;
                const double teacher_most = terms[4], per = kLog2eD / a.temperature;
                // (the exponent in 64 bits, its fraction's power by the hardware: the library's 64-bit routine costs a wavefront a SIMD in registers)
                auto prob = [&](int j) {
                    const double d = ((double)logit_of(a.teacher, a.teacher_dtype, row * a.k + j) - teacher_most) * per, whole = rint(d);
                    return d < -160.0 ? 0.0f : terms[5] * ldexpf(__builtin_amdgcn_exp2f((float)(d - whole)), (int)whole);
                };
                const float f = Elem<T>::widen(x[e - e0]);
                float q = prob(j);
                bool is_first = true;
                if (twice) {  // an index twice: the first adds up the others
                    for (int l = 0; l < j && is_first; ++l) is_first = token(l) != e;
                    for (int l = j + 1; l < a.k && is_first; ++l)
                        if (token(l) == e) q += prob(l);
                }
                const float y = terms[1] * exp_of(f - terms[0], a.steps);
                if (is_first) out[e - e0] = Elem<T>::narrow(w * (y - q));
            }
        }
        auto grad = [&](T v) {
            const float f = Elem<T>::widen(v);
            return Elem<T>::narrow(coef * exp_of(f - rest_most, a.steps));
        };
        auto is_named = [&](int e) { return on && bits[(e + shift) >> 5] >> ((e + shift) & 31) & 1; };
        if (lane < head && !is_named(lane)) out[lane] = on ? grad(first) : first;
        if (lane < n - tail && !is_named(tail + lane)) out[tail + lane] = on ? grad(last) : last;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int v = lane + i * 64;
            if (v >= vecs) continue;
            const int e = head + v * VEC;
            uint32_t some = 0;
            if (on) {
#pragma unroll
                for (int l = 0; l < VEC; ++l) p[i].v[l] = grad(p[i].v[l]);
                some = bits[(e + shift) >> 5] >> ((e + shift) & 31) & ((1u << VEC) - 1);
            }
            if (some == 0) store_pack_stream<T, VEC>(out + e, p[i]);
            else
#pragma unroll
                for (int l = 0; l < VEC; ++l)
                    if (!(some >> l & 1)) out[e + l] = p[i].v[l];
        }
        fence();
    }
}

}  // namespace

// (us of loss alone, bf16 [8192, 50257] with the rest, rows whole, in two, four and eight parts: 186, 213, 245, 313)
int distill_split(int dtype, int64_t rows, int64_t cols) {
    if (rows == 0 || rows > 2047) return 1;
    const int64_t bytes = cols * (int64_t)dtype_size(dtype);
    return (int)std::max<int64_t>(1, std::min<int64_t>({64, 4096 / rows, bytes / (16 << 10)}));
}

void launch_distill_loss(int dtype, const DistillArgs& a, hipStream_t st) {
    if (a.rows > 0)
        HPT_WITH_TYPE(dtype, {
            const unsigned blocks = (unsigned)std::min<int64_t>(a.rows * a.split, 1 << 20);
            if (a.teacher_lse) distill_stats_kernel<T, true><<<blocks, kThreads, 0, st>>>(a);
            else distill_stats_kernel<T, false><<<blocks, kThreads, 0, st>>>(a);
            // (a launch has fewer than 2^32 work items. Walked by the kernel, 49 registers would spill: f32 [100000, 64] 384 -> 631 us)
            constexpr int64_t most = (int64_t)kRowsAtOnce << 20;
            for (int64_t from = 0; from < a.rows; from += most)
                distill_rows_kernel<T><<<(unsigned)((std::min(most, a.rows - from) + kRowsAtOnce - 1) / kRowsAtOnce), 64 * kRowsAtOnce, 0, st>>>(a, from);
        });
    distill_sum_kernel<<<1, 1024, 0, st>>>(a);
}

void launch_distill_loss_backward(int dtype, const DistillGradArgs& a, hipStream_t st) {
    HPT_WITH_TYPE(dtype, {
        constexpr int VEC = 16 / sizeof(T);
        const int most = 64 * kGradVecs * VEC;
        const int pieces = (a.cols + most - 1) / most;
        const int each = ((a.cols + pieces - 1) / pieces + VEC - 1) / VEC * VEC;
        const int64_t blocks = (a.rows * pieces + kThreads / 64 - 1) / (kThreads / 64);
        distill_grad_kernel<T><<<(unsigned)std::min<int64_t>(blocks, 1 << 20), kThreads, 0, st>>>(a, pieces, each);
    });
}

}  // namespace hpt
