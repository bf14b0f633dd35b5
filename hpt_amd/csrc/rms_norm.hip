// RMS norm over rows: h = x (+ residual), y = h / sqrt(mean(h^2) + eps) * gamma, y in the inputs' type or in 8 bits with scales; and
// its backward pass.
//
// Backward, with r = 1 / sqrt(mean(x^2) + eps) and c = sum over the row of gy * gamma * x:
//   gx = r * gy * gamma - x * r^3 * c / cols (+ what else arrives at x),   ggamma = sum over the rows of gy * x * r.
// r and c come from the one read of x and gy that the result needs anyway.
//
// Everything here is bound by memory: a row is read once into the registers of the threads that share it and written once (longer rows are swept). Sums
// are f32 (x of two bytes widened exactly, squares and products in f32), of rows that are swept f64 from vector to vector; h is rounded to the inputs' type first, as a
// separate addition would have stored it, and y is computed from the rounded h; y is rounded once.
#include <algorithm>

#include "block_rows.hpp"

namespace hpt {

namespace {

// 8-bit outputs: value = y / scale, scale = the group's largest |y| over the type's largest value. 2^-120 at least, so that its
// reciprocal exists (a row of zeros); a group with a NaN gets a NaN for scale.
constexpr float kLeastScale = 0x1p-120f;

template <int Q> __device__ __forceinline__ float group_scale(uint32_t most_bits) {
    const float most = __uint_as_float(most_bits);
    const float s = most / (Q == QUANT_I8 ? 127.0f : 448.0f);
    return s < kLeastScale ? kLeastScale : s;
}
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// VEC values over their scale, in 8 bits each: the f32 quotient, to nearest, ties to even. |y / s| is no more than the type's largest value times 1 + 2^-23, which rounds to that
// value in both types; NaN becomes 0 in i8 and NaN in e4m3. The product with a float reciprocal is up to 1.5 places off the quotient, and what lies beside a border between two codes
// would fall to its wrong side: the reciprocal comes in two pieces, which leave 2^-22 of a place. The second is never negative, so that -0 stays -0, and no subnormal up to scales of 2^60.
// us, one piece and two: bf16 [13107, 5120] 45.6 and 49.2, with a residual by 128 [8192, 4096] 40.4 and 41.1.
template <int Q, int VEC> __device__ __forceinline__ Pack<uint8_t, VEC> quantized(const float (&y)[VEC], float s) {
    static_assert(VEC % 4 == 0, "four values to a word");
    union { uint32_t w[VEC / 4]; Pack<uint8_t, VEC> p; } u;
    float q[VEC];
    if (s <= 0x1p60f) {
        float inv = 1.0f / s, rest = fmaf(-s, inv, 1.0f);
        if (rest < 0.0f) {
            inv = __uint_as_float(__float_as_uint(inv) - 1);
            rest = fmaf(-s, inv, 1.0f);
        }
        const float low = rest * inv;
#pragma unroll
        for (int i = 0; i < VEC; ++i) q[i] = fmaf(y[i], inv, y[i] * low);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) q[i] = y[i] / s;
    }
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
        if constexpr (Q == QUANT_E4M3) {
            int w = 0;
            w = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i], q[4 * i + 1], w, false);
            w = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i + 2], q[4 * i + 3], w, true);
            u.w[i] = (uint32_t)w;
        } else {
            uint32_t w = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float v = q[4 * i + k];
                const int n = v == v ? (int)__builtin_rintf(v) : 0;
                w |= ((uint32_t)n & 0xffu) << (8 * k);
            }
            u.w[i] = w;
        }
    }
    return u.p;
}
template <int Q> __device__ __forceinline__ uint8_t quantized_one(float y, float s) {
    const float v[4] = {y, 0.0f, 0.0f, 0.0f};
    return quantized<Q, 4>(v, s).v[0];
}

// Whether workgroups walk the rows with the next one on its way while a row is summed and written, or take a row each and leave it to their
// number that memory is busy. us, a row each -> walked: one operand f16 [13107, 5120] 64 -> 50, bf16 [4096, 16384] 65 -> 50, [8190, 4097]
// 32 -> 27, [16384, 4096] 50.4 -> 49.7; in 8 bits bf16 [13107, 5120] 73.2 -> 49.3, [16384, 4096] 51.7 -> 42.6, f32 [8192, 2048] 22.4 -> 20.1; x + residual in 8 bits f16 [13107, 5120] 80.7 -> 77.7, bf16 [8192, 8192]
// 77.5 -> 75.0, but [8192, 4096] 38.7 -> 41.1 and [16384, 4096] 73.0 -> 78.0. x + residual in its own type is ahead without ([16384, 4096] 89 against 97, [13107, 5120]
// 89 against 99), and beyond 16 elements per thread a second row does not fit the registers.
template <class T, int NC, bool RES, int Q> constexpr bool kAhead = (!RES || Q != QUANT_NONE) && NC * 16 / (int)sizeof(T) <= 16;

// Rows held in registers; gamma is fetched once. x + residual f16 [13107, 5120] 90 us, 6.0 TB/s of two reads and two writes; in 8 bits by 128 bf16 [8192, 4096]
// 46 us, 5.1 TB/s; a step of decoding, bf16 [8, 4096], 4.5 us, a launch and the latency of one row. Q: groups of `group` elements are `group` / VEC neighbouring lanes
// (a power of two of them, within a wavefront), or the whole row.
template <class T, int NC, bool AL, bool RES, int Q>
__global__ __launch_bounds__(1024) void rms_row_kernel(const RmsArgs a) {
    constexpr int VEC = 16 / sizeof(T);
    using At = Slot<VEC, AL>;
    __shared__ float sums[2 * 16];
    __shared__ uint32_t mosts[2 * 16];
    int turn = 0, turn_most = 0;
    const int tpr = a.tpr, lane = threadIdx.x % tpr, ty = threadIdx.x / tpr, rpb = blockDim.x / tpr;
    Pack<T, VEC> g[NC];
    if (a.gamma) {
#pragma unroll
        for (int k = 0; k < NC; ++k) g[k] = load_slot<T, AL>((const T*)a.gamma, At(lane + k * tpr, a.cols));
#pragma unroll
        for (int k = 0; k < NC; ++k) clean_slot<T, AL>(g[k], At(lane + k * tpr, a.cols));
    }
    const int64_t step = (int64_t)gridDim.x * rpb;
    Pack<T, VEC> p[NC], q[RES ? NC : 1];
    auto fetch = [&](int64_t row) {
        const int cols = row < a.rows ? a.cols : 0;  // (threads behind the last row go along to the barriers)
        const T* x = (const T*)a.x + (cols ? offset_of(a.kept, row) : 0);
#pragma unroll
        for (int k = 0; k < NC; ++k) p[k] = load_slot<T, AL>(x, At(lane + k * tpr, cols));
        if constexpr (RES) {
#pragma unroll
            for (int k = 0; k < NC; ++k) q[k] = load_slot<T, AL>((const T*)a.res + row * a.cols, At(lane + k * tpr, cols));
        }
    };
    if constexpr (kAhead<T, NC, RES, Q>) fetch((int64_t)blockIdx.x * rpb + ty);
    for (int64_t first = (int64_t)blockIdx.x * rpb; first < a.rows; first += step) {
        const int64_t row = first + ty;
        const int cols = row < a.rows ? a.cols : 0;
        if constexpr (!kAhead<T, NC, RES, Q>) fetch(row);
        Pack<T, VEC> h[NC];
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            h[k] = p[k];
            if constexpr (RES) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) h[k].v[i] = Elem<T>::narrow(Elem<T>::widen(p[k].v[i]) + Elem<T>::widen(q[k].v[i]));
            }
            clean_slot<T, AL>(h[k], At(lane + k * tpr, cols));
        }
        if constexpr (kAhead<T, NC, RES, Q>) {
            if (first + step < a.rows) fetch(row + step);
        }
        if constexpr (RES) {
            if (a.sum) {
#pragma unroll
                for (int k = 0; k < NC; ++k) store_slot<T, VEC, AL>((T*)a.sum + row * a.cols, At(lane + k * tpr, cols), h[k]);
            }
        }
        float ss[1] = {0.0f};
#pragma unroll
        for (int k = 0; k < NC; ++k) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) ss[0] = fmaf(Elem<T>::widen(h[k].v[i]), Elem<T>::widen(h[k].v[i]), ss[0]);
        }
        fold_row<SumF>(ss, tpr, sums, turn);
        const float r = 1.0f / sqrtf(ss[0] / (float)a.cols + a.eps);
        auto value = [&](int k, float (&y)[VEC]) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) y[i] = a.gamma ? Elem<T>::widen(h[k].v[i]) * r * Elem<T>::widen(g[k].v[i]) : Elem<T>::widen(h[k].v[i]) * r;
        };
        if constexpr (Q == QUANT_NONE) {
            T* out = (T*)a.out + row * a.cols;
#pragma unroll
            for (int k = 0; k < NC; ++k) {
                float y[VEC];
                value(k, y);
                Pack<T, VEC> o;
#pragma unroll
                for (int i = 0; i < VEC; ++i) o.v[i] = Elem<T>::narrow(y[i]);
                store_slot<T, VEC, AL>(out, At(lane + k * tpr, cols), o);
            }
        } else {
            uint8_t* out = (uint8_t*)a.out + row * a.cols;
            // (places that hold no element are zeros: 0 * r is NaN where r is infinite or NaN, and then every element of the row is NaN too)
            uint32_t m[NC];
#pragma unroll
            for (int k = 0; k < NC; ++k) {
                float y[VEC];
                value(k, y);
                m[k] = 0;
#pragma unroll
                for (int i = 0; i < VEC; ++i) m[k] = MaxBits::comb(m[k], magnitude(y[i]));
            }
            if (a.group == a.cols) {
                uint32_t all[1] = {0};
#pragma unroll
                for (int k = 0; k < NC; ++k) all[0] = MaxBits::comb(all[0], m[k]);
                fold_row<MaxBits>(all, tpr, mosts, turn_most);
                const float s = group_scale<Q>(all[0]);
                if (lane == 0 && cols) a.scale[row] = s;
#pragma unroll
                for (int k = 0; k < NC; ++k) m[k] = __float_as_uint(s);
            } else {
                const int lanes = a.group / VEC;
#pragma unroll
                for (int k = 0; k < NC; ++k) {
                    const float s = group_scale<Q>(group_reduce<MaxBits>(m[k], lanes));
                    const int v = lane + k * tpr;
                    if ((lane & (lanes - 1)) == 0 && v * VEC < cols) a.scale[row * (a.cols / a.group) + v / lanes] = s;
                    m[k] = __float_as_uint(s);
                }
            }
#pragma unroll
            for (int k = 0; k < NC; ++k) {
                float y[VEC];
                value(k, y);
                store_slot<uint8_t, VEC, AL>(out, At(lane + k * tpr, cols), quantized<Q, VEC>(y, __uint_as_float(m[k])));
            }
        }
    }
}

// Any row length and any group: a workgroup of 1024 sweeps a row twice (8-bit output with one scale per row: three times). With a
// residual the first sweep stores the sum where the caller wants it, and later sweeps read it there: x or the residual may be that very
// memory. A thread meets the same vectors in every sweep, but for the groups, which wavefronts take by elements behind a barrier.
template <class T, bool RES, int Q>
__global__ __launch_bounds__(1024) void rms_stream_kernel(const RmsArgs a) {
    constexpr int VEC = 16 / sizeof(T);
    __shared__ double sums[2 * 16];
    __shared__ uint32_t mosts[2 * 16];
    int turn = 0, turn_most = 0;
    const int vecs = (a.cols + VEC - 1) / VEC;
    const T* gamma = (const T*)a.gamma;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = (const T*)a.x + offset_of(a.kept, row);
        const T* res = RES ? (const T*)a.res + row * a.cols : nullptr;
        T* sum = RES && a.sum ? (T*)a.sum + row * a.cols : nullptr;
        double ss[1] = {0.0};
        for (int v = threadIdx.x; v < vecs; v += 1024) {
            Pack<T, VEC> p = sweep_vec<T>(x, v, a.cols);
            if constexpr (RES) {
                const Pack<T, VEC> q = sweep_vec<T>(res, v, a.cols);
#pragma unroll
                for (int i = 0; i < VEC; ++i) p.v[i] = Elem<T>::narrow(Elem<T>::widen(p.v[i]) + Elem<T>::widen(q.v[i]));
                if (sum) store_sweep_vec<T, VEC>(sum, v, a.cols, p);
            }
            float add = 0.0f;
#pragma unroll
            for (int i = 0; i < VEC; ++i) add = fmaf(Elem<T>::widen(p.v[i]), Elem<T>::widen(p.v[i]), add);
            ss[0] += add;
        }
        fold_row<SumD>(ss, 1024, sums, turn);
        const float r = 1.0f / sqrtf((float)(ss[0] / a.cols) + a.eps);
        const T* h = sum ? sum : x;
        const bool add = RES && !sum;
        auto value = [&](int e) {
            float v = Elem<T>::widen(h[e]);
            if (add) v = Elem<T>::widen(Elem<T>::narrow(v + Elem<T>::widen(res[e])));
            v *= r;
            return gamma ? v * Elem<T>::widen(gamma[e]) : v;
        };
        auto values = [&](int v, float (&y)[VEC]) {
            Pack<T, VEC> p = sweep_vec<T>(h, v, a.cols);
            if (add) {
                const Pack<T, VEC> q = sweep_vec<T>(res, v, a.cols);
#pragma unroll
                for (int i = 0; i < VEC; ++i) p.v[i] = Elem<T>::narrow(Elem<T>::widen(p.v[i]) + Elem<T>::widen(q.v[i]));
            }
            Pack<T, VEC> g;
            if (gamma) g = sweep_vec<T>(gamma, v, a.cols);
#pragma unroll
            for (int i = 0; i < VEC; ++i) y[i] = gamma ? Elem<T>::widen(p.v[i]) * r * Elem<T>::widen(g.v[i]) : Elem<T>::widen(p.v[i]) * r;
        };
        if constexpr (Q == QUANT_NONE) {
            for (int v = threadIdx.x; v < vecs; v += 1024) {
                float y[VEC];
                values(v, y);
                Pack<T, VEC> p;
#pragma unroll
                for (int i = 0; i < VEC; ++i) p.v[i] = Elem<T>::narrow(y[i]);
                store_sweep_vec<T, VEC>((T*)a.out + row * a.cols, v, a.cols, p);
            }
        } else {
            uint8_t* out = (uint8_t*)a.out + row * a.cols;
            if (a.group == a.cols) {
                uint32_t m[1] = {0};
                for (int v = threadIdx.x; v < vecs; v += 1024) {
                    float y[VEC];
                    values(v, y);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) m[0] = MaxBits::comb(m[0], magnitude(y[i]));
                }
                fold_row<MaxBits>(m, 1024, mosts, turn_most);
                const float s = group_scale<Q>(m[0]);
                if (threadIdx.x == 0) a.scale[row] = s;
                for (int v = threadIdx.x; v < vecs; v += 1024) {
                    float y[VEC];
                    values(v, y);
                    store_sweep_vec<uint8_t, VEC>(out, v, a.cols, quantized<Q, VEC>(y, s));
                }
            } else {
                __syncthreads();  // the sums that other threads have stored
                const int groups = a.cols / a.group, l = threadIdx.x & 63;
                for (int n = threadIdx.x >> 6; n < groups; n += 16) {
                    uint32_t m = 0;
                    for (int e = l; e < a.group; e += 64) m = MaxBits::comb(m, magnitude(value(n * a.group + e)));
                    const float s = group_scale<Q>(group_reduce<MaxBits>(m, 64));
                    if (l == 0) a.scale[row * groups + n] = s;
                    for (int e = l; e < a.group; e += 64) out[n * a.group + e] = quantized_one<Q>(value(n * a.group + e), s);
                }
            }
        }
    }
}

bool on_grid(const void* p) { return ((uintptr_t)p & 15) == 0; }
// Rows of whole vectors that all start on the vector grid.
bool rows_on_grid(const void* p, const Dims& kept, int vec) {
    bool ok = on_grid(p);
    for (int i = 0; i < kept.n; ++i) ok = ok && (kept.size[i] == 1 || kept.stride[i] % vec == 0);
    return ok;
}

template <class T, bool RES, int Q> void launch_of(const RmsArgs& given, hipStream_t st) {
    constexpr int VEC = 16 / sizeof(T);
    RmsArgs a = given;
    // (eight vectors of f32 and of a residual spill: [1024, 30001] 128 us, streamed 114)
    constexpr int most = sizeof(T) == 4 ? (RES ? 6 : 8) : 4;
    const bool al = a.cols % VEC == 0 && rows_on_grid(a.x, a.kept, VEC) && on_grid(a.res) && on_grid(a.gamma) && on_grid(a.sum) && on_grid(a.out);
    const bool grouped = Q != QUANT_NONE && a.group != a.cols;
    // lanes of a group: a power of two of them within a wavefront
    const int lanes = grouped && a.group % VEC == 0 ? a.group / VEC : 0;
    const bool by_lanes = !grouped || (al && lanes >= 1 && lanes <= 64 && (lanes & (lanes - 1)) == 0);
    const RowDeal d = deal_row(a.cols, sizeof(T), 2, most, grouped && by_lanes ? lanes : 1);
    if (!d.held() || !by_lanes || a.cols < VEC) {
        rms_stream_kernel<T, RES, Q><<<(unsigned)std::min<int64_t>(a.rows, 1 << 16), 1024, 0, st>>>(a);
        return;
    }
    a.tpr = d.tpr;
    const int64_t blocks = (a.rows + d.rows_per_block() - 1) / d.rows_per_block();
    // walked: as many workgroups as run at once, of six wavefronts on each SIMD, with a residual four (24 -> 16 wavefronts per compute unit: bf16
    // [8192, 8192] in 8 bits 96 -> 84 us, without a residual 46 -> 51)
    const int64_t resident = 256 * std::max(1, (RES ? 16 : 24) / (d.threads / 64));
    HPT_WITH_NC(d.nc, {
        constexpr int N = NC > most ? most : NC;
        const unsigned grid = (unsigned)std::min<int64_t>(blocks, kAhead<T, N, RES, Q> ? resident : 1 << 16);
        if (al) rms_row_kernel<T, N, true, RES, Q><<<grid, d.threads, 0, st>>>(a);
        else rms_row_kernel<T, N, false, RES, Q><<<grid, d.threads, 0, st>>>(a);
    });
}

// ---- backward -------------------------------------------------------------------------------------

// Rows held in registers; each workgroup walks rows and keeps its sums for gamma in registers, which leave as one row of partial sums. Bound by memory:
// bf16 [16384, 4096] with a third operand 103 us, 5.2 TB/s, and 5 us for the columns; f32 [1237, 1001] 7 and 4 us, two launches and their latency.
template <class T, int NC, bool AL, bool MORE>
__global__ __launch_bounds__(1024) void rms_grad_kernel(const RmsGradArgs a) {
    constexpr int VEC = 16 / sizeof(T);
    using At = Slot<VEC, AL>;
    __shared__ float sums[2 * 16 * 2];
    extern __shared__ float fold[];  // several rows per workgroup: [cols]
    int turn = 0;
    const int tpr = a.tpr, lane = threadIdx.x % tpr, ty = threadIdx.x / tpr, rpb = blockDim.x / tpr;
    Pack<T, VEC> g[NC];
    if (a.gamma) {
#pragma unroll
        for (int k = 0; k < NC; ++k) g[k] = load_slot<T, AL>((const T*)a.gamma, At(lane + k * tpr, a.cols));
#pragma unroll
        for (int k = 0; k < NC; ++k) clean_slot<T, AL>(g[k], At(lane + k * tpr, a.cols));
    }
    float acc[NC][VEC] = {};
    for (int64_t first = (int64_t)blockIdx.x * rpb; first < a.rows; first += (int64_t)gridDim.x * rpb) {
        const int64_t row = first + ty;
        const int cols = row < a.rows ? a.cols : 0;
        const T* xr = (const T*)a.x + (cols ? offset_of(a.kept, row) : 0);
        Pack<T, VEC> x[NC], gy[NC], more[MORE ? NC : 1];
#pragma unroll
        for (int k = 0; k < NC; ++k) x[k] = load_slot<T, AL>(xr, At(lane + k * tpr, cols));
#pragma unroll
        for (int k = 0; k < NC; ++k) gy[k] = load_slot<T, AL>((const T*)a.gy + row * a.cols, At(lane + k * tpr, cols));
        if constexpr (MORE) {
#pragma unroll
            for (int k = 0; k < NC; ++k) more[k] = load_slot<T, AL>((const T*)a.gsum + row * a.cols, At(lane + k * tpr, cols));
        }
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            clean_slot<T, AL>(x[k], At(lane + k * tpr, cols));
            clean_slot<T, AL>(gy[k], At(lane + k * tpr, cols));
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float xv = Elem<T>::widen(x[k].v[i]);
                float gv = Elem<T>::widen(gy[k].v[i]);
                if (a.gamma) gv *= Elem<T>::widen(g[k].v[i]);
                s[0] = fmaf(xv, xv, s[0]);
                s[1] = fmaf(gv, xv, s[1]);
            }
        }
        fold_row<SumF>(s, tpr, sums, turn);
        const float r = 1.0f / sqrtf(s[0] / (float)a.cols + a.eps);
        const float c = r * (r * (s[1] / (float)a.cols));  // (r^2 alone may be beyond f32)
        T* gx = (T*)a.gx + row * a.cols;
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            const At at(lane + k * tpr, cols);
            Pack<T, VEC> p;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float xv = Elem<T>::widen(x[k].v[i]), gv = Elem<T>::widen(gy[k].v[i]);
                const float gg = a.gamma ? gv * Elem<T>::widen(g[k].v[i]) : gv;
                float d = r * (gg - xv * c);
                if constexpr (MORE) d += Elem<T>::widen(more[k].v[i]);
                p.v[i] = Elem<T>::narrow(d);
                acc[k][i] = fmaf(gv, xv * r, acc[k][i]);  // (without a row x and gy are zeros and r finite: eps > 0)
            }
            store_slot<T, VEC, AL>(gx, at, p);
        }
    }
    if (!a.ggamma) return;
    float* part = a.partial + (int64_t)blockIdx.x * a.cols;
    if (rpb == 1) {
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            const At at(lane + k * tpr, a.cols);
            if (at.lo == 0) {
                __builtin_memcpy(part + at.s, acc[k], sizeof acc[k]);
            } else if constexpr (!AL) {
#pragma unroll
                for (int i = 1; i < VEC; ++i)
                    if (i >= at.lo) part[at.s + i] = acc[k][i];
            }
        }
        return;
    }
    // The rows that share a wavefront by their lanes, then the wavefronts one after the other: the same order always. (All rows one after the other, 32 of them:
    // bf16 [577, 90] 27 us, so 9.6, [131072, 64] 29.5 and 17.3.)
    for (int w = tpr; w < 64; w <<= 1) {
#pragma unroll
        for (int k = 0; k < NC; ++k) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[k][i] += __shfl_xor(acc[k][i], w, 64);
        }
    }
    for (int t = 0; t < (int)blockDim.x >> 6; ++t) {
        if (t == (int)threadIdx.x >> 6 && (threadIdx.x & 63) < (unsigned)tpr) {
#pragma unroll
            for (int k = 0; k < NC; ++k) {
                const At at(lane + k * tpr, a.cols);
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    if (i >= at.lo) fold[at.s + i] = t == 0 ? acc[k][i] : fold[at.s + i] + acc[k][i];
            }
        }
        __syncthreads();
    }
    for (int e = threadIdx.x; e < a.cols; e += blockDim.x) part[e] = fold[e];
}

// Rows of any length, swept twice; the sums for gamma grow in the workgroup's own row of partial sums (a thread meets its own elements). Rows shorter than a vector can be
// many thousands for each workgroup: the first thread keeps their sums in f64 (in f32, 4096 rows of the same sign were 5e-5 off).
template <class T>
__global__ __launch_bounds__(1024) void rms_grad_stream_kernel(const RmsGradArgs a) {
    constexpr int VEC = 16 / sizeof(T);
    __shared__ double sums[2 * 16 * 2];
    int turn = 0;
    const int vecs = (a.cols + VEC - 1) / VEC;
    const T* gamma = (const T*)a.gamma;
    float* part = a.ggamma ? a.partial + (int64_t)blockIdx.x * a.cols : nullptr;
    bool fresh = true;
    double few[VEC] = {};
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, fresh = false) {
        const T* x = (const T*)a.x + offset_of(a.kept, row);
        const T* gy = (const T*)a.gy + row * a.cols;
        const T* gsum = a.gsum ? (const T*)a.gsum + row * a.cols : nullptr;
        double s[2] = {0.0, 0.0};
        for (int v = threadIdx.x; v < vecs; v += 1024) {
            const Pack<T, VEC> xp = sweep_vec<T>(x, v, a.cols), gp = sweep_vec<T>(gy, v, a.cols);
            Pack<T, VEC> g;
            if (gamma) g = sweep_vec<T>(gamma, v, a.cols);
            float add[2] = {0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float xv = Elem<T>::widen(xp.v[i]);
                float gv = Elem<T>::widen(gp.v[i]);
                if (gamma) gv *= Elem<T>::widen(g.v[i]);
                add[0] = fmaf(xv, xv, add[0]);
                add[1] = fmaf(gv, xv, add[1]);
            }
            s[0] += add[0];
            s[1] += add[1];
        }
        fold_row<SumD>(s, 1024, sums, turn);
        const float r = 1.0f / sqrtf((float)(s[0] / a.cols) + a.eps);
        const float c = r * (r * (float)(s[1] / a.cols));
        for (int v = threadIdx.x; v < vecs; v += 1024) {
            const Pack<T, VEC> xp = sweep_vec<T>(x, v, a.cols), gp = sweep_vec<T>(gy, v, a.cols);
            Pack<T, VEC> g, more, p;
            if (gamma) g = sweep_vec<T>(gamma, v, a.cols);
            if (gsum) more = sweep_vec<T>(gsum, v, a.cols);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float xv = Elem<T>::widen(xp.v[i]), gv = Elem<T>::widen(gp.v[i]);
                const float gg = gamma ? gv * Elem<T>::widen(g.v[i]) : gv;
                float d = r * (gg - xv * c);
                if (gsum) d += Elem<T>::widen(more.v[i]);
                p.v[i] = Elem<T>::narrow(d);
                const int e = v * VEC + i;
                if (vecs == 1) few[i] += gv * (xv * r);
                else if (part && e < a.cols) part[e] = fresh ? gv * (xv * r) : part[e] + gv * (xv * r);
            }
            store_sweep_vec<T, VEC>((T*)a.gx + row * a.cols, v, a.cols, p);
        }
    }
    if (part && vecs == 1 && threadIdx.x == 0) {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (i < a.cols) part[i] = (float)few[i];
    }
}

// The partial sums of gamma's gradient, column by column: 32 columns and 32 rows at a time, in a fixed order, summed in f64.
__global__ __launch_bounds__(1024) void rms_grad_columns_kernel(const float* partial, int64_t parts, int cols, float* out) {
    __shared__ double meet[32][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    for (int first = blockIdx.x * 32; first < cols; first += gridDim.x * 32) {
        const int col = first + tx;
        double s = 0;
        if (col < cols) {
#pragma unroll 8
            for (int64_t p = ty; p < parts; p += 32) s += partial[p * cols + col];
        }
        __syncthreads();  // (the columns before have been read)
        meet[ty][tx] = s;
        __syncthreads();
        if (ty == 0 && col < cols) {
            for (int k = 1; k < 32; ++k) s += meet[k][tx];
            out[col] = (float)s;
        }
    }
}

// Two vectors per thread, four of f32: with more the accumulators spill. `more`: a third operand. With it a row of two-byte elements goes to four or
// to eight wavefronts: of five (a second one on one of the four SIMDs) fewer workgroups run at once: us, bf16 [13107, 5120] 184 with 320 threads, 141 with 512,
// but 90 against 112 without a third operand, where three workgroups of five wavefronts have room.
// Two-byte rows above a wavefront have one vector per thread while each workgroup has few rows to walk, up to 48 MiB, of longer ones 16 MiB: us, bf16 [6000, 1608] 29 with two, 25
// with one, [1500, 2353] 19 and 17, [500, 5120] 13.3 and 11.1, but [12000, 4096] 65 and 77.
RowDeal grad_deal(int dtype, int64_t rows, int64_t cols, bool more) {
    const bool wide = dtype == HPT_F32;
    const int64_t vecs = (cols * (int64_t)dtype_size(dtype) + 15) / 16;
    const bool one = !wide && vecs > 128 && vecs <= 1024 && rows * vecs <= (int64_t)(vecs <= 256 ? 3 : 1) << 20;
    RowDeal d = deal_row(cols, dtype_size(dtype), one ? 1 : 2, wide ? 4 : 2);
    if (!wide && more && d.nc > 1 && d.threads > 256 && d.threads < 512) d.tpr = d.threads = 512;
    return d;
}
// As many workgroups as run at once; in more, the last round is mostly empty, in fewer, memory waits. That is four wavefronts on each SIMD of two-byte
// elements, five (`five`) of bf16 without a third operand in whole, aligned vectors where a row has four at most (f16 takes more registers: [51392, 640] 55 in 1024, 77
// in 1280; bf16 [20000, 513] off the grid 26 and 33): us, bf16 [16384, 4096] and a third operand 512 workgroups 170, 768 125, 1024 108,
// 1280 145; [16384, 4096] without 86 in 1024, 82 in 1280. Of f32 three and two are enough, and more meet in memory: [32768, 1024] and a third operand 99 in 1024, 105
// in 2048, [16384, 2048] 98 in 512, 105 in 1024.
// Few rows: near two to a workgroup, each of which leaves a row of partial sums, and the same on every compute unit: f32 [1237, 1001] 12.0 in 512, 12.6 in 618,
// 11.5 in 768, 13.7 in 1237.
int64_t grad_parts(int dtype, int64_t rows, int64_t cols, bool more, bool five) {
    const RowDeal d = grad_deal(dtype, rows, cols, more);
    const int64_t blocks = (rows + d.rows_per_block() - 1) / d.rows_per_block();
    const int waves = d.threads / 64;
    const int64_t resident = 256 * (dtype == HPT_F32 ? std::max(2, (more ? 8 : 12) / waves) : std::max(1, (five && waves <= 4 ? 20 : 16) / waves));
    // (256 MiB of partial sums at most, or one row of them where that is longer: from 32 Mi columns on a single workgroup walks the rows)
    return std::min({blocks, resident, std::max<int64_t>(512, blocks * 5 / 8 / 256 * 256), std::max<int64_t>(1, (64 << 20) / std::max<int64_t>(1, cols))});
}

}  // namespace

void launch_rms_norm(int dtype, int quant, const RmsArgs& a, hipStream_t st) {
    HPT_WITH_TYPE(dtype, {
        if (quant == QUANT_I8) a.res ? launch_of<T, true, QUANT_I8>(a, st) : launch_of<T, false, QUANT_I8>(a, st);
        else if (quant == QUANT_E4M3) a.res ? launch_of<T, true, QUANT_E4M3>(a, st) : launch_of<T, false, QUANT_E4M3>(a, st);
        else a.res ? launch_of<T, true, QUANT_NONE>(a, st) : launch_of<T, false, QUANT_NONE>(a, st);
    });
}

// (The caller of a workspace's size does not say whether there is a third operand.)
int64_t rms_grad_partials(int dtype, int64_t rows, int64_t cols) { return std::max(grad_parts(dtype, rows, cols, false, true), grad_parts(dtype, rows, cols, true, false)); }

void launch_rms_norm_backward(int dtype, const RmsGradArgs& given, hipStream_t st) {
    RmsGradArgs a = given;
    const RowDeal d = grad_deal(dtype, a.rows, a.cols, a.gsum);
    const int vec = 16 / (int)dtype_size(dtype);
    const bool al = a.cols % vec == 0 && rows_on_grid(a.x, a.kept, vec) && on_grid(a.gy) && on_grid(a.gsum) && on_grid(a.gamma) && on_grid(a.gx);
    const int64_t parts = grad_parts(dtype, a.rows, a.cols, a.gsum, al && !a.gsum && dtype == HPT_BF16);  // (no rows: none, and gamma's gradient is zeros)
    a.tpr = d.tpr;
    const size_t lds = d.rows_per_block() > 1 ? (size_t)a.cols * 4 : 0;
    if (parts) HPT_WITH_TYPE(dtype, {
        constexpr int VEC = 16 / sizeof(T);
        if (!d.held() || a.cols < VEC) {
            rms_grad_stream_kernel<T><<<(unsigned)parts, 1024, 0, st>>>(a);
        } else {
            HPT_WITH_NC(d.nc, {
                constexpr int M = sizeof(T) == 4 ? (NC > 4 ? 4 : NC) : (NC > 2 ? 2 : NC);
                if (al && a.gsum) rms_grad_kernel<T, M, true, true><<<(unsigned)parts, d.threads, lds, st>>>(a);
                else if (al) rms_grad_kernel<T, M, true, false><<<(unsigned)parts, d.threads, lds, st>>>(a);
                else if (a.gsum) rms_grad_kernel<T, M, false, true><<<(unsigned)parts, d.threads, lds, st>>>(a);
                else rms_grad_kernel<T, M, false, false><<<(unsigned)parts, d.threads, lds, st>>>(a);
            });
        }
    });
    if (a.ggamma) rms_grad_columns_kernel<<<std::min((a.cols + 31) / 32, 1 << 16), 1024, 0, st>>>(a.partial, parts, a.cols, a.ggamma);
}

}  // namespace hpt
