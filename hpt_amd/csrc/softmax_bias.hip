// Attention's softmax(scale * scores + table[bucket(key - query), head]) over the keys, and its backward pass.
//
// The bias depends on key - query alone, and from the distance on at which the last bucket begins (`far`) on nothing: a workgroup
// that works on one head keeps it in LDS by distance, -far ... far, and takes the two ends for all that lies beyond. Masks are
// parameters (causal, and the lengths of a padded batch): a row keeps the keys up to a last one, what lies behind is neither read
// nor computed, its results are zeros, and so is a row that keeps no key.
//
// Backward, from the probabilities p and the gradient g that arrives at them: d = p (g - sum over the keys of p g); the scores' gradient
// is scale * d, the table's the sum of d over all places of a bucket. Those sums are taken by distance first: within a row every
// distance below `far` occurs once, so a row adds to its places in LDS without a conflict, and the threads keep the sums of the
// two ends in registers. Rows follow one another, workgroups leave a row of partial sums each, which a second kernel folds: the
// order is the same always.
//
// Bound by memory: one read of every live score, one write of every result (longer rows are swept twice). Sums and maxima f32, sums of rows that are swept f64 from
// vector to vector; results rounded once.
#include <algorithm>
#include <cmath>

#include "block_rows.hpp"

namespace hpt {

Buckets make_buckets(int64_t total, bool both, int64_t max_distance) {
    if (total < 2 || total > kMostBuckets) fail(HPT_ERR_PARAM, "position bias: %lld buckets, outside 2..%d", (long long)total, kMostBuckets);
    if (both && total % 2) fail(HPT_ERR_PARAM, "position bias: an odd number of buckets (%lld) for two directions", (long long)total);
    Buckets b;
    b.both = both;
    b.n = (int)(both ? total / 2 : total);
    if (b.n < 2) fail(HPT_ERR_PARAM, "position bias: each direction needs two buckets at least");
    const int half = b.n / 2;  // of one distance each
    if (max_distance <= half || max_distance > kMostDistance)
        fail(HPT_ERR_PARAM, "position bias: max_distance %lld outside %d..%d for %d buckets a direction", (long long)max_distance, half + 1, kMostDistance, b.n);
    for (int k = 0; k <= half; ++k) b.begin[k] = (uint16_t)k;
    // bucket half + j begins at the first whole distance not below half * (max_distance / half)^(j / (n - half)); a power that comes
    // within 1e-9 of a whole number is taken for it (doubles are off by 1e-14 or so after up to 127 products)
    const double step = std::pow((double)max_distance / half, 1.0 / (b.n - half));
    double at = half;
    for (int j = 1; half + j < b.n; ++j) {
        at *= step;
        b.begin[half + j] = (uint16_t)std::ceil(at * (1 - 1e-9));
    }
    b.far = b.begin[b.n - 1];
    std::fill(b.begin + b.n, b.begin + kMostBuckets, (uint16_t)0xffff);
    return b;
}

namespace {

// (Counted along `begin`, eight at a time, which every lane reads at the same place: a search would wait for one load after the other.)
__device__ __forceinline__ int bucket_of(const Buckets& b, int d) {
    typedef uint32_t Eight __attribute__((ext_vector_type(4), may_alias));
    const int far = d < 0 ? -d : b.both ? d : 0, first = b.n / 2 & ~7;  // below it a bucket is its distance
    int k = min(far, first - 1);
#pragma unroll 2
    for (int j = first; j < b.n; j += 8) {
        const Eight e = *(const Eight*)(b.begin + j);
#pragma unroll
        for (int i = 0; i < 4; ++i) k += ((int)(e[i] & 0xffff) <= far) + ((int)(e[i] >> 16) <= far);
    }
    return k + (d > 0 && b.both ? b.n : 0);
}
// Places by distance in LDS: -far ... right, and a vector's length more on both sides, so that a vector that reaches into the range, from
// either side, has all its places there. Where keys ahead of the query share bucket 0, one place is enough for them and for distance 0.
constexpr int kPad = 8;
__device__ __forceinline__ int right_of(const Buckets& b) { return b.both ? b.far : 0; }
__host__ __device__ inline int places_of(const Buckets& b) { return b.far + (b.both ? b.far : 0) + 1 + 2 * kPad; }

// What the rows of a matrix have in common: how many keys its sequence has, and the position of its query q0. Beyond +-2^30 every key is
// far or hidden, as there are fewer than 2^29 of them (and distances stay within 32 bits).
struct Place {
    int length, pos;
    template <class A> __device__ __forceinline__ Place(const A& a, int64_t matrix, int64_t q0) {
        int64_t n = a.keys;
        if (a.lengths) {
            const int64_t b = quotient(matrix, a.heads);
            const int64_t len = a.lengths64 ? ((const int64_t*)a.lengths)[b] : (int64_t)((const int32_t*)a.lengths)[b];
            n = len < 0 ? 0 : len < n ? len : n;
        }
        length = (int)n;
        const int64_t p = q0 + a.offset, most = 1 << 30;
        pos = (int)(p > most ? most : p < -most ? -most : p);
    }
    // The end of the keys that query q0 + i sees.
    __device__ __forceinline__ int live(int i, int causal) const { return causal ? max(min(length, pos + i + 1), 0) : length; }
};

template <class T> __device__ __forceinline__ void fill_bias(const BiasArgs& a, int64_t head, float* bias) {
    const int n = places_of(a.buckets), right = right_of(a.buckets);
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int d = min(max(i - kPad - a.buckets.far, -a.buckets.far), right);
        bias[i] = Elem<T>::widen(((const T*)a.table)[bucket_of(a.buckets, d) * a.table_bucket + head * a.table_head]);
    }
}

// VEC scores from key e on -> scale * x + bias, -inf from key `live` on and before place lo. Where no lane of
// the wavefront is near the query the two ends of the bias are all that is needed, otherwise all take them from LDS, the
// far ones from its padding.
template <class T, int VEC>
__device__ __forceinline__ void biased(const Pack<T, VEC>& p, int e, int lo, int live, int pos, float scale, int far, int right, const float* bias, float (&s)[VEC]) {
    const int d = e - pos;
    if (__any(d > -far - VEC && d < right)) {
        const float* b = bias + (min(max(d, -far - kPad), right) + far + kPad);
#pragma unroll
        for (int i = 0; i < VEC; ++i) s[i] = fmaf(scale, Elem<T>::widen(p.v[i]), b[i]);
    } else {
        const float b = bias[d >= right ? far + right + kPad : 0];
#pragma unroll
        for (int i = 0; i < VEC; ++i) s[i] = fmaf(scale, Elem<T>::widen(p.v[i]), b);
    }
    if (lo > 0 || e + VEC > live) {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (i < lo || e + i >= live) s[i] = -__builtin_huge_valf();
    }
}

// Rows held in registers. An item is `per_item` rows of one matrix; the first row is on its way while the bias comes together, every other
// one while the row before it is summed and written. bf16 [8, 16, 1024, 1024] with lengths 90 us, 5.0 TB/s: next to memory, the bias by distance and an
// exponential for every element. One query, f16 [16, 32, 1, 4097], 7.8 us: bias, loads, two folds and the store follow one another.
template <class T, int NC, bool AL>
__global__ __launch_bounds__(1024, NC <= 2 ? 5 : 4) void bias_row_kernel(const BiasArgs a) {
    constexpr int VEC = 16 / sizeof(T);
    using At = Slot<VEC, AL>;
    extern __shared__ float bias[];
    __shared__ float most[2 * 16], sums[2 * 16];
    int turn_m = 0, turn_s = 0;
    const int tpr = a.tpr, lane = threadIdx.x % tpr, ty = threadIdx.x / tpr, rpb = blockDim.x / tpr;
    const int far = a.buckets.far, right = right_of(a.buckets);
    for (int64_t item = blockIdx.x; item < a.items; item += gridDim.x) {
        const int64_t matrix = quotient(item, a.chunks), q0 = (item - matrix * a.chunks) * a.per_item;
        const int n = (int)min((int64_t)a.per_item, a.queries - q0);  // rows
        const Place place(a, matrix, q0);
        const T* x0 = (const T*)a.x + offset_of(a.matrices, matrix) + q0 * a.query_stride;
        T* out0 = (T*)a.out + (matrix * a.queries + q0) * a.keys;
        Pack<T, VEC> p[NC];
        auto fetch = [&](int i) {
            const int live = i < n ? place.live(i, a.causal) : 0;
            const T* x = x0 + i * a.query_stride;
#pragma unroll
            for (int k = 0; k < NC; ++k) {
                At at(lane + k * tpr, a.keys);
                if (at.s + at.lo >= live) at.lo = VEC;  // (nothing of it is live: not read)
                p[k] = load_slot<T, AL>(x, at);
            }
        };
        fetch(ty);
        __syncthreads();  // (the bias of the item before is no longer read)
        fill_bias<T>(a, matrix - quotient(matrix, a.heads) * a.heads, bias);
        __syncthreads();
        for (int first = 0; first < n; first += rpb) {
            const int i = first + ty;
            const int live = i < n ? place.live(i, a.causal) : 0, pos = place.pos + i;
            float s[NC][VEC];
            float m[1] = {-__builtin_huge_valf()};
#pragma unroll
            for (int k = 0; k < NC; ++k) {
                const At at(lane + k * tpr, a.keys);
                biased<T, VEC>(p[k], at.s, at.lo, live, pos, a.scale, far, right, bias, s[k]);
#pragma unroll
                for (int j = 0; j < VEC; ++j) m[0] = fmaxf(m[0], s[k][j]);
            }
            if (first + rpb < n) fetch(i + rpb);
            fold_row<MaxF>(m, tpr, most, turn_m);
            // (a hidden place is -inf and its exponential 0: in a row of nothing else, too)
            const float base = m[0] == -__builtin_huge_valf() ? 0.0f : m[0];
            float t[1] = {0.0f};
            // (two-byte types: one multiply-add makes the hardware's argument; what rounding base * log2 e costs is in every term and in their
            // sum alike. It is 2^-4 at most while the row's largest score is within 2^20, but beyond some 1e9 it leaves the exponential's range: rows that a caller has
            // masked as a whole with a large finite number take the differences, which are exact where they matter.)
            if (sizeof(T) == 2 && fabsf(base) < 0x1p20f) {
                constexpr float kLog2e = 1.44269504f;
                const float shift = -base * kLog2e;
#pragma unroll
                for (int k = 0; k < NC; ++k) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        s[k][j] = __builtin_amdgcn_exp2f(fmaf(s[k][j], kLog2e, shift));
                        t[0] += s[k][j];
                    }
                }
            } else {
#pragma unroll
                for (int k = 0; k < NC; ++k) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        s[k][j] = exp_row<T>(s[k][j] - base);
                        t[0] += s[k][j];
                    }
                }
            }
            fold_row<SumF>(t, tpr, sums, turn_s);
            const float inv = live ? 1.0f / t[0] : 0.0f;
            const bool number = t[0] > 0.0f || !live;
            if (i < n) {
                T* out = out0 + (int64_t)i * a.keys;
#pragma unroll
                for (int k = 0; k < NC; ++k) {
                    const At at(lane + k * tpr, a.keys);
                    Pack<T, VEC> o;
#pragma unroll
                    for (int j = 0; j < VEC; ++j) o.v[j] = Elem<T>::narrow(s[k][j] * inv);
                    if (__any(!number)) {  // keys of -inf alone, or a NaN or +inf among them: the hidden ones are zeros all the same
#pragma unroll
                        for (int j = 0; j < VEC; ++j) o.v[j] = number ? o.v[j] : Elem<T>::narrow(at.s + j < live ? __builtin_nanf("") : 0.0f);
                    }
                    store_slot<T, VEC, AL>(out, at, o);
                }
            }
        }
    }
}

// (maximum, sum of exponentials below it) of what has been seen, and of two such.
template <class T, class S> __device__ __forceinline__ void meet(float& m, S& s, float m2, S s2) {
    const float n = fmaxf(m, m2);
    // (nothing seen is (-inf, 0); equal infinities are no distance apart; a NaN is in its sum)
    s = s * (S)(m == n ? 1.0f : exp_row<T>(m - n)) + s2 * (S)(m2 == n ? 1.0f : exp_row<T>(m2 - n));
    m = n;
}

// Statistics of the live keys of `row` from vector v0 to v1, over the whole workgroup (a multiple of 64 threads).
template <class T> __device__ __forceinline__ void sweep_stats(const BiasArgs& a, const T* x, int v0, int v1, int live, int pos, const float* bias, float* most, double* sums, float& m, float& total) {
    constexpr int VEC = 16 / sizeof(T);
    m = -__builtin_huge_valf();
    double s = 0.0;
    for (int v = v0 + threadIdx.x; v < v1 && v * VEC < live; v += blockDim.x) {
        float t[VEC];
        biased<T, VEC>(sweep_vec<T>(x, v, a.keys), v * VEC, 0, live, pos, a.scale, a.buckets.far, right_of(a.buckets), bias, t);
        float n = m;
#pragma unroll
        for (int i = 0; i < VEC; ++i) n = fmaxf(n, t[i]);
        float add = 0.0f;
#pragma unroll
        for (int i = 0; i < VEC; ++i) add += v * VEC + i >= live ? 0.0f : t[i] == n ? 1.0f : exp_row<T>(t[i] - n);
        s = (m == n ? s : s * (double)exp_row<T>(m - n)) + (double)add;
        m = n;
    }
#pragma unroll
    for (int w = 1; w < 64; w <<= 1) meet<T>(m, s, __shfl_xor(m, w, 64), shfl_xor_any(s, w));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        most[threadIdx.x >> 6] = m;
        sums[threadIdx.x >> 6] = s;
    }
    __syncthreads();
    m = most[0];
    s = sums[0];
    for (int w = 1; w < (int)blockDim.x >> 6; ++w) meet<T>(m, s, most[w], sums[w]);
    total = (float)s;
}

template <class T> __device__ __forceinline__ void sweep_apply(const BiasArgs& a, const T* x, T* out, int v0, int v1, int live, int pos, const float* bias, float m, float s) {
    constexpr int VEC = 16 / sizeof(T);
    // (a row that keeps keys of -inf alone, or one of +inf, is NaN, as any softmax's)
    const bool none = m == -__builtin_huge_valf() || m == __builtin_huge_valf();
    const float inv = none ? __builtin_nanf("") : 1.0f / s;
    for (int v = v0 + threadIdx.x; v < v1; v += blockDim.x) {
        Pack<T, VEC> o;
        if (v * VEC < live) {
            float t[VEC];
            biased<T, VEC>(sweep_vec<T>(x, v, a.keys), v * VEC, 0, live, pos, a.scale, a.buckets.far, right_of(a.buckets), bias, t);
#pragma unroll
            for (int i = 0; i < VEC; ++i) o.v[i] = Elem<T>::narrow(v * VEC + i >= live ? 0.0f : exp_row<T>(t[i] - m) * inv);
        } else {
            __builtin_memset(&o, 0, sizeof o);
        }
        store_sweep_vec<T, VEC>(out, v, a.keys, o);
    }
}

// Rows of any length, a workgroup each: statistics, then a second read.
template <class T>
__global__ __launch_bounds__(1024) void bias_stream_kernel(const BiasArgs a) {
    constexpr int VEC = 16 / sizeof(T);
    extern __shared__ float bias[];
    __shared__ float most[16];
    __shared__ double sums[16];
    const int vecs = (a.keys + VEC - 1) / VEC;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const int64_t matrix = quotient(row, a.queries), q = row - matrix * a.queries;
        __syncthreads();
        fill_bias<T>(a, matrix - quotient(matrix, a.heads) * a.heads, bias);
        __syncthreads();
        const Place place(a, matrix, q);
        const int live = place.live(0, a.causal), pos = place.pos;
        const T* x = (const T*)a.x + offset_of(a.matrices, matrix) + q * a.query_stride;
        float m, s;
        sweep_stats<T>(a, x, 0, vecs, live, pos, bias, most, sums, m, s);
        sweep_apply<T>(a, x, (T*)a.out + row * a.keys, 0, vecs, live, pos, bias, m, s);
    }
}

// Few, long rows: a.split workgroups share one. APPLY: the second launch, in which each folds all parts' statistics.
template <class T, bool APPLY>
__global__ __launch_bounds__(256) void bias_split_kernel(const BiasArgs a) {
    constexpr int VEC = 16 / sizeof(T);
    extern __shared__ float bias[];
    __shared__ float most[4];
    __shared__ double sums[4];
    const int64_t row = blockIdx.x / (unsigned)a.split, matrix = quotient(row, a.queries), q = row - matrix * a.queries;
    const int part = blockIdx.x % a.split;
    const int vecs = (a.keys + VEC - 1) / VEC, each = (vecs + a.split - 1) / a.split;
    const int v0 = min(part * each, vecs), v1 = min(v0 + each, vecs);
    fill_bias<T>(a, matrix - quotient(matrix, a.heads) * a.heads, bias);
    __syncthreads();
    const Place place(a, matrix, q);
    const int live = place.live(0, a.causal), pos = place.pos;
    const T* x = (const T*)a.x + offset_of(a.matrices, matrix) + q * a.query_stride;
    float m, s;
    if constexpr (!APPLY) {
        sweep_stats<T>(a, x, v0, v1, live, pos, bias, most, sums, m, s);
        if (threadIdx.x == 0) {
            a.partial[2 * (row * a.split + part)] = m;
            a.partial[2 * (row * a.split + part) + 1] = s;
        }
    } else {
        const float* p = a.partial + 2 * row * a.split;
        m = p[0];
        s = p[1];
        for (int k = 1; k < a.split; ++k) meet<T>(m, s, p[2 * k], p[2 * k + 1]);
        sweep_apply<T>(a, x, (T*)a.out + row * a.keys, v0, v1, live, pos, bias, m, s);
    }
}

// ---- backward -------------------------------------------------------------------------------------

// By how much the places of rows at position `pos` are shifted, and the quadruples of an array with room for any shift.
__device__ __forceinline__ int shift_of(const Buckets& b, int pos) { return (pos - b.far - kPad) & 3; }
__host__ __device__ inline int quads_of(const Buckets& b) { return (places_of(b) + 3 + 3) / 4; }

typedef float Quad __attribute__((ext_vector_type(4), may_alias));

// (Rows that are swept.) What a row's VEC elements from key e on add: to the places of their distances, or, beyond `far` and `right`, to the thread's own sums of
// the ends. Hidden elements are zeros. Rows add to a place one after the other, each once, so that the sums do not depend on any order
// though the LDS adds by itself.
template <int VEC>
__device__ __forceinline__ void add_by_distance(const float (&d)[VEC], int e, int pos, int far, int right, float* places, double& left_end, double& right_end) {
    const int r = e - pos;
    if (r > -far - VEC && r < right) {
        float* at = places + (r + far + kPad);
#pragma unroll
        for (int i = 0; i < VEC; ++i) __hip_atomic_fetch_add(at + i, d[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    } else {
        float s = d[0];
#pragma unroll
        for (int i = 1; i < VEC; ++i) s += d[i];
        if (r < 0) left_end += s;
        else right_end += s;
    }
}

// The workgroup's sums by distance -> by bucket, into its row of partial sums; eight lanes share a bucket. `places`: arrays of `length`, number g for
// rows at positions pos + g modulo 4. They become one first, each place by a thread that alone reads it in all of them (without that step, f16 [32, 12, 64, 64] 11.1 us, with it
// 10.1; unrolled further it costs the rows' loop registers). Every thread of the workgroup comes here.
template <class Op, class A> __device__ __forceinline__ void leave_buckets(const Buckets& b, float* places, int arrays, int length, int pos, A left_end, A right_end, float* out) {
    __shared__ A ends[2 * 16 * 2];
    const int total = b.both ? 2 * b.n : b.n, zero = b.far + kPad;
    A e[2] = {left_end, right_end};
    int turn = 0;
    fold_row<Op>(e, blockDim.x, ends, turn);
    __syncthreads();  // (a single wavefront has passed none in the fold)
    const int shift = shift_of(b, pos);
    if (arrays > 1) {
        for (int q = threadIdx.x; q < places_of(b); q += blockDim.x) {
            float s = places[q + shift];
#pragma unroll 2
            for (int g = 1; g < arrays; ++g) s += places[g * length + q + shift_of(b, pos + g)];
            places[q + shift] = s;
        }
        __syncthreads();
    }
    const int part = threadIdx.x & 7;
    for (int k = threadIdx.x >> 3; k < total; k += blockDim.x >> 3) {
        const bool ahead = b.both && k >= b.n;
        const int j = ahead ? k - b.n : k;
        // distances of bucket k: of its direction's last one also those of the margin; bucket 0 of a single direction has the other's margin
        const int from = ahead && j == 0 ? 1 : !b.both && j == 0 ? -kPad : b.begin[j], to = j + 1 < b.n ? min((int)b.begin[j + 1], b.far + kPad + 1) : b.far + kPad + 1;
        float s = part == 0 && j == b.n - 1 ? (float)e[ahead] : 0.0f;
        if (part == 0 && !b.both && j == 0) s += (float)e[1];
        for (int d = from + part; d < to; d += 8)
            s += places[(ahead ? zero + d : zero - d) + shift];
        s = group_reduce<SumF>(s, 8);
        if (part == 0) out[k] = s;
    }
}

// Rows held in registers, one after the other into the same places. The rows that meet in one array of places all stand at the same position
// modulo 4 (four rows side by side or more have an array each, longer ones are dealt to four in turn), and the array is shifted by what that
// is, so that a vector's places are whole aligned quadruples: read, added to and written with 128-bit accesses that meet no bank
// twice. (By single words, eight to a vector, every instruction met each bank eight times: 73 us of bf16 [16, 16, 256, 256] were theirs.)
// Rows above a wavefront pass a barrier between two rows' additions (the fold); rows within one are kept in order by the fence.
// bf16 [4, 16, 1024, 1024], causal, 61 us, 4.4 TB/s, and 4 us for the table; next to memory, the additions in LDS.
template <class T, int NC, bool AL>
__global__ __launch_bounds__(1024, NC <= 2 ? (AL ? 6 : 5) : 4) void bias_grad_kernel(const BiasGradArgs a) {
    constexpr int VEC = 16 / sizeof(T);
    using At = Slot<VEC, AL>;
    extern __shared__ __attribute__((aligned(16))) float places[];  // [arrays, quads]
    __shared__ float sums[2 * 16];
    int turn = 0;
    const int tpr = a.tpr, lane = threadIdx.x % tpr, ty = threadIdx.x / tpr, rpb = blockDim.x / tpr;
    const int far = a.buckets.far, right = right_of(a.buckets), quads = quads_of(a.buckets), arrays = max(rpb, 4);
    for (int64_t item = blockIdx.x; item < a.items; item += gridDim.x) {
        const int64_t matrix = quotient(item, a.chunks), q0 = (item - matrix * a.chunks) * a.per_item;
        const int n = (int)min((int64_t)a.per_item, a.queries - q0);  // rows
        const Place place(a, matrix, q0);
        const int64_t at0 = (matrix * a.queries + q0) * a.keys;
        float left_end = 0.0f, right_end = 0.0f;
        Pack<T, VEC> pp[NC], gp[NC];
        __syncthreads();  // (the item before has left its sums)
        for (int i = threadIdx.x; i < quads * arrays; i += blockDim.x) ((Quad*)places)[i] = Quad{0.0f, 0.0f, 0.0f, 0.0f};
        __syncthreads();
        for (int first = 0; first < n; first += rpb) {
            const int i = first + ty;
            const int live = i < n ? place.live(i, a.causal) : 0, pos = place.pos + i;
            const T *p = (const T*)a.p + at0 + (int64_t)i * a.keys, *g = (const T*)a.g + at0 + (int64_t)i * a.keys;
#pragma unroll
            for (int k = 0; k < NC; ++k) {
                At at(lane + k * tpr, a.keys);
                if (at.s + at.lo >= live) at.lo = VEC;  // (nothing of it is live: not read)
                pp[k] = load_slot<T, AL>(p, at);
                gp[k] = load_slot<T, AL>(g, at);
            }
            float s[1] = {0.0f};
#pragma unroll
            for (int k = 0; k < NC; ++k) {
                const At at(lane + k * tpr, a.keys);
                clean_slot<T, AL>(pp[k], at);
                clean_slot<T, AL>(gp[k], at);
                if (at.s + VEC > live) {  // the last live vector: hidden elements become zeros
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        if (at.s + j >= live) pp[k].v[j] = gp[k].v[j] = Elem<T>::narrow(0.0f);
                    }
                }
#pragma unroll
                for (int j = 0; j < VEC; ++j) s[0] = fmaf(Elem<T>::widen(pp[k].v[j]), Elem<T>::widen(gp[k].v[j]), s[0]);
            }
            fold_row<SumF>(s, tpr, sums, turn);
            const bool finite = fabsf(s[0]) < __builtin_huge_valf();
            T* out = (T*)a.out + at0 + (int64_t)i * a.keys;
            float* mine = places + (rpb >= 4 ? ty : i & 3) * 4 * quads;
            const int shift = far + kPad - pos + shift_of(a.buckets, pos);  // of a key's place: a multiple of 4 for keys that are
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int k = 0; k < NC; ++k) {
                const At at(lane + k * tpr, a.keys);
                float d[VEC];
                Pack<T, VEC> o;
#pragma unroll
                for (int j = 0; j < VEC; ++j) d[j] = Elem<T>::widen(pp[k].v[j]) * (Elem<T>::widen(gp[k].v[j]) - s[0]);
                if (__any(!finite)) {  // (0 * (0 - s) would be NaN in hidden places)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) d[j] = finite || (j >= at.lo && at.s + j < live) ? d[j] : 0.0f;
                }
#pragma unroll
                for (int j = 0; j < VEC; ++j) o.v[j] = Elem<T>::narrow(a.scale * d[j]);
                if (i < n) store_slot<T, VEC, AL>(out, at, o);
                if (!a.table_grad || at.s + at.lo >= live) continue;
                const int r = at.s - pos;
                if (r <= -far - VEC || r >= right) {
                    float t = d[0];
#pragma unroll
                    for (int j = 1; j < VEC; ++j) t += d[j];
                    if (r < 0) left_end += t;
                    else right_end += t;
                } else if (AL || at.lo == 0) {
                    Quad* to = (Quad*)(mine + at.s + shift);
#pragma unroll
                    for (int j = 0; j < VEC / 4; ++j) to[j] += Quad{d[4 * j], d[4 * j + 1], d[4 * j + 2], d[4 * j + 3]};
                } else {  // the row's last vector, taken from its end backwards: its own elements by words
#pragma unroll
                    for (int j = 1; j < VEC; ++j) {
                        if (j >= at.lo) mine[at.s + shift + j] += d[j];
                    }
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        if (a.table_grad) leave_buckets<SumF>(a.buckets, places, arrays, 4 * quads, place.pos, left_end, right_end, a.partial + item * (a.buckets.both ? 2 * a.buckets.n : a.buckets.n));
    }
}

// Rows of any length: two sweeps.
template <class T>
__global__ __launch_bounds__(1024) void bias_grad_stream_kernel(const BiasGradArgs a) {
    constexpr int VEC = 16 / sizeof(T);
    extern __shared__ float places[];
    __shared__ double sums[2 * 16];
    int turn = 0;
    const int far = a.buckets.far, right = right_of(a.buckets), n = places_of(a.buckets), vecs = (a.keys + VEC - 1) / VEC;
    for (int64_t item = blockIdx.x; item < a.items; item += gridDim.x) {
        const int64_t matrix = quotient(item, a.chunks), q0 = (item - matrix * a.chunks) * a.per_item;
        const int64_t q1 = q0 + a.per_item < a.queries ? q0 + a.per_item : a.queries;
        double left_end = 0.0, right_end = 0.0;
        __syncthreads();  // (the item before has left its sums)
        for (int i = threadIdx.x; i < n; i += 1024) places[i] = 0.0f;
        __syncthreads();
        for (int64_t q = q0; q < q1; ++q) {
            const int64_t row = matrix * a.queries + q;
            const Place place(a, matrix, q);
            const int live = place.live(0, a.causal), pos = place.pos;
            const T *p = (const T*)a.p + row * a.keys, *g = (const T*)a.g + row * a.keys;
            double fold[1] = {0.0};
            for (int v = threadIdx.x; v * VEC < live; v += 1024) {
                const Pack<T, VEC> pp = sweep_vec<T>(p, v, a.keys), gp = sweep_vec<T>(g, v, a.keys);
                float add = 0.0f;
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    if (v * VEC + i < live) add = fmaf(Elem<T>::widen(pp.v[i]), Elem<T>::widen(gp.v[i]), add);
                fold[0] += add;
            }
            fold_row<SumD>(fold, 1024, sums, turn);  // (its barrier also keeps two rows' additions apart)
            const float s = (float)fold[0];
            for (int v = threadIdx.x; v < vecs; v += 1024) {
                float d[VEC];
                Pack<T, VEC> o;
                __builtin_memset(&o, 0, sizeof o);
                if (v * VEC < live) {
                    const Pack<T, VEC> pp = sweep_vec<T>(p, v, a.keys), gp = sweep_vec<T>(g, v, a.keys);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        d[i] = v * VEC + i < live ? Elem<T>::widen(pp.v[i]) * (Elem<T>::widen(gp.v[i]) - s) : 0.0f;
                        o.v[i] = Elem<T>::narrow(a.scale * d[i]);
                    }
                    if (a.table_grad) add_by_distance<VEC>(d, v * VEC, pos, far, right, places, left_end, right_end);
                }
                store_sweep_vec<T, VEC>((T*)a.out + row * a.keys, v, a.keys, o);
            }
        }
        if (a.table_grad) leave_buckets<SumD>(a.buckets, places, 1, 0, far + kPad, left_end, right_end, a.partial + item * (a.buckets.both ? 2 * a.buckets.n : a.buckets.n));
    }
}

// The table's gradient [buckets, heads]: a wavefront for each entry folds the items of its head in a fixed order, in f64.
__global__ __launch_bounds__(256) void bias_grad_table_kernel(const float* partial, int64_t matrices, int64_t chunks, int64_t heads, int buckets, float* out) {
    const int64_t items = quotient(matrices, heads) * chunks;
    for (int64_t entry = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); entry < heads * buckets; entry += (int64_t)gridDim.x * 4) {
        const int64_t bucket = quotient(entry, heads), head = entry - bucket * heads;
        double s = 0;
        for (int64_t i = threadIdx.x & 63; i < items; i += 64) {
            const int64_t batch = quotient(i, chunks);  // (item i of this head is item batch * heads * chunks + head * chunks + i % chunks of all)
            s += partial[((batch * (heads - 1) + head) * chunks + i) * buckets + bucket];
        }
#pragma unroll
        for (int w = 1; w < 64; w <<= 1) s += shfl_xor_any(s, w);
        if ((threadIdx.x & 63) == 0) out[entry] = (float)s;
    }
}
void launch_table(const BiasGradArgs& a, int64_t matrices, hipStream_t st) {
    const int buckets = a.buckets.both ? 2 * a.buckets.n : a.buckets.n;
    const unsigned grid = (unsigned)std::min<int64_t>((a.heads * buckets + 3) / 4, 1 << 20);
    bias_grad_table_kernel<<<grid, 256, 0, st>>>(a.partial, matrices, a.chunks, a.heads, buckets, a.table_grad);
}

// Distances that no query and key have need no place: `far` as if the last bucket began right behind the largest there is. (256 distances both ways, backward, bf16
// [40, 32, 45, 45] 23.3 us, so 15.6.)
Buckets within_reach(Buckets b, int64_t queries, int64_t keys, int64_t offset) {
    const int64_t behind = queries - 1 + offset, ahead = b.both ? keys - 1 - offset : 0;
    b.far = (int)std::min<int64_t>(b.far, std::max<int64_t>({behind, ahead, 0}) + 1);
    return b;
}

bool on_grid(const void* p) { return ((uintptr_t)p & 15) == 0; }

size_t bias_lds(const Buckets& b) { return (size_t)places_of(b) * 4; }

// Four vectors per thread: a row's maximum and sum cost the same for two. us of two vectors per thread and of up to four, f16 [8, 16, 512, 520] (65 vectors) 42.4 and 31.5, [.., 1032]
// 77.3 and 53.3, and alike for 1024 keys, 45.2.
// Rows above a wavefront go to workgroups of 128, 256, 512 or 768 threads with three or four vectors each (f32 four to eight): a fifth wavefront shares a
// SIMD with the first, and then fewer workgroups run at once. us, f16 [8, 16, 256, 4104] 320 threads of two vectors 148, 256 of three 109; [1, 16, 256, 8208] 576 of two 55, 512
// of three 41; [4, 16, 256, 6144] 384 of two 98, 256 of three 63; one query, [64, 32, 1, 4104] 320 of two 20.1, 256 of three 14.1; f32 [4, 16, 256, 4400] 320 of four 117, 256 of five 96.
// (385 ... 512 two-byte vectors: of whole matrices, [8, 16, 256, 4096], 256 threads of two 83, 128 of four 109; of one query, [64, 32, 1, 4096], 12.2 and 9.7.)
// A workgroup holds rows of one matrix: where that has few (a step of decoding has one), they get the lanes of a wavefront (f32 [128, 16, 1, 256] 6.1 with 64, 7.4 with 16),
// and the workgroup is no larger than they need. Up to four rows of one query for each compute unit get up to four wavefronts, as the latency of a row is
// all there is: f16 [16, 32, 1, 2048] 6.0 with 256 threads, 7.0 with 64, f32 [16, 32, 1, 1000] 5.9 and 6.9; f16 [128, 16, 1, 1536] 7.5 with 64, 8.6 with 128.
RowDeal bias_deal(int dtype, int64_t rows, int64_t queries, int64_t keys) {
    const bool wide = dtype == HPT_F32;
    const int64_t vecs = (keys * (int64_t)dtype_size(dtype) + 15) / 16;
    RowDeal d = deal_row(keys, dtype_size(dtype), 4, most_vecs(dtype));
    if (!d.held()) return d;
    if (d.tpr > 64) {
        const int64_t fit[] = {wide ? 512 : queries == 1 ? 512 : 384, wide ? 1536 : 1024, wide ? 4096 : 2048, wide ? 0 : 2304};
        const int threads[] = {128, 256, 512, 768};
        d.tpr = 1024;
        for (int i = 3; i >= 0; --i)
            if (vecs <= fit[i]) d.tpr = threads[i];
        d.threads = d.tpr;
    }
    while (d.tpr < 64 && queries * d.tpr < 64) d.tpr *= 2;
    if (queries == 1 && rows <= 1024 && d.tpr < 256 && vecs > 64) d.tpr = d.threads = (int)std::min<int64_t>(256, (vecs + 63) / 64 * 64);
    d.nc = (int)((vecs + d.tpr - 1) / d.tpr);
    while (d.tpr <= 64 && d.threads > 64 && d.threads / 2 >= queries * d.tpr) d.threads /= 2;
    return d;
}
// Backward: two vectors per thread of two operands, four of f32 (two-byte elements with four: us, bf16 [8, 16, 256, 520] 27.3 with two and 34.0, [.., 4096] 158 and 207), but one for 129 ...
// 256 vectors, where two would leave a third of the lanes idle or so (us of one and of two, [.., 1200] 49.5 and 55.4, [.., 1536] 59.6 and 65.7, [.., 2048] 70.9 and 77.1). 32 rows side
// by side at most, because each of them has places of its own. 768 threads are three wavefronts on each SIMD: [1, 16, 256, 9600] with 640 threads 57.8, with 768 51.8; f32 [1, 16, 256, 8196] with 576 87, with 768 71.
RowDeal bias_grad_deal(int dtype, int64_t keys) {
    const bool wide = dtype == HPT_F32;
    const int64_t vecs = (keys * (int64_t)dtype_size(dtype) + 15) / 16;
    RowDeal d = deal_row(keys, dtype_size(dtype), wide ? 4 : vecs > 128 && vecs <= 256 ? 1 : 2, wide ? 4 : 2, 8);
    if (d.held() && d.threads > 512 && d.threads < 768) {
        d.tpr = d.threads = 768;
        d.nc = (int)((vecs + 767) / 768);
    }
    return d;
}
// Rows of a matrix that a workgroup takes one after the other, in rounds of those side by side: 96 KiB of operands and results for 256 threads
// (each workgroup fetches its bias or clears its places first), 64 rows at most, but so that there are 512 workgroups. us, forward / backward, for 64, 96 and 128 KiB: bf16 [4, 16, 1024, 1024], causal, 52 / 69, 49 / 65, 58 / 67, [2, 16, 2048, 2048], causal,
// 112 / 147, 105 / 124, 103 / 126, [8, 16, 1024, 1024] 93 / 151, 96 / 141, 98 / 144. [16, 16, 256, 256] with 1024 workgroups 14.1 / 24.6, with 4096
// 18.9 / 30.8.
int64_t rounds_of(int64_t rows, const RowDeal& d, int64_t row_bytes) {
    return std::max<int64_t>(1, std::min<int64_t>({(int64_t)384 * d.threads / row_bytes, 64, rows / 512}) / d.rows_per_block());
}

}  // namespace

// Rows that registers do not hold, and few of them, are split into parts of 16 KiB at least: two launches, but on more compute units. (Rows that
// registers hold stay whole: bf16 [32, 32768] 9.9 us against 13.9 split, [256, 32768] 12.6 against 19.)
int bias_split(int dtype, int64_t rows, int64_t keys) {
    if (rows == 0 || rows >= 512 || deal_row(keys, dtype_size(dtype), 1, most_vecs(dtype)).held()) return 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>({64, 1024 / rows, keys * (int64_t)dtype_size(dtype) / (16 << 10)}));
}

void launch_softmax_bias(int dtype, const BiasArgs& given, hipStream_t st) {
    BiasArgs a = given;
    a.buckets = within_reach(a.buckets, a.queries, a.keys, a.offset);
    const size_t lds = bias_lds(a.buckets);
    const int64_t matrices = a.rows / a.queries;
    HPT_WITH_TYPE(dtype, {
        constexpr int VEC = 16 / sizeof(T);
        const RowDeal d = bias_deal(dtype, a.rows, a.queries, a.keys);
        if (a.split > 1) {
            const unsigned grid = (unsigned)(a.rows * a.split);
            bias_split_kernel<T, false><<<grid, 256, lds, st>>>(a);
            bias_split_kernel<T, true><<<grid, 256, lds, st>>>(a);
        } else if (!d.held() || a.keys < VEC) {
            bias_stream_kernel<T><<<(unsigned)std::min<int64_t>(a.rows, 1 << 16), 1024, lds, st>>>(a);
        } else {
            a.tpr = d.tpr;
            a.per_item = (int)(rounds_of(a.rows, d, 2 * a.keys * (int64_t)sizeof(T)) * d.rows_per_block());
            a.chunks = (a.queries + a.per_item - 1) / a.per_item;
            a.items = matrices * a.chunks;
            bool al = a.keys % VEC == 0 && on_grid(a.x) && on_grid(a.out) && (a.queries == 1 || a.query_stride % VEC == 0);
            for (int i = 0; i < a.matrices.n; ++i) al = al && (a.matrices.size[i] == 1 || a.matrices.stride[i] % VEC == 0);
            const unsigned grid = (unsigned)std::min<int64_t>(a.items, 1 << 20);
            HPT_WITH_NC(d.nc, {
                if (al) bias_row_kernel<T, NC, true><<<grid, d.threads, lds, st>>>(a);
                else bias_row_kernel<T, NC, false><<<grid, d.threads, lds, st>>>(a);
            });
        }
    });
}

int64_t bias_grad_items(int dtype, int64_t matrices, int64_t queries, int64_t keys, int* per_item) {
    const RowDeal d = bias_grad_deal(dtype, keys);
    *per_item = (int)(rounds_of(matrices * queries, d, 3 * keys * (int64_t)dtype_size(dtype)) * d.rows_per_block());
    return matrices * ((queries + *per_item - 1) / *per_item);
}

void launch_softmax_bias_backward(int dtype, const BiasGradArgs& given, hipStream_t st) {
    BiasGradArgs a = given;
    if (a.rows == 0) {  // a table's gradient of zeros
        a.chunks = 1;
        launch_table(a, 0, st);
        return;
    }
    a.buckets = within_reach(a.buckets, a.queries, a.keys, a.offset);
    const int64_t matrices = a.rows / a.queries;
    a.items = bias_grad_items(dtype, matrices, a.queries, a.keys, &a.per_item);
    a.chunks = (a.queries + a.per_item - 1) / a.per_item;
    RowDeal d = bias_grad_deal(dtype, a.keys);
    const bool held = d.held();
    const size_t one = bias_lds(a.buckets);
    // (far buckets take more LDS: fewer rows side by side, the same items)
    const size_t array = (size_t)quads_of(a.buckets) * 16;
    while (d.tpr < 64 && array * d.rows_per_block() > (20 << 10)) d.tpr *= 2;
    const size_t lds = array * std::max(4, d.rows_per_block());
    d.nc = (int)(((int64_t)a.keys * (int64_t)dtype_size(dtype) + 16 * d.tpr - 1) / (16 * d.tpr));
    a.tpr = d.tpr;
    const unsigned grid = (unsigned)std::min<int64_t>(a.items, 1 << 20);
    HPT_WITH_TYPE(dtype, {
        constexpr int VEC = 16 / sizeof(T);
        const bool al = a.keys % VEC == 0 && on_grid(a.p) && on_grid(a.g) && on_grid(a.out);
        if (!held || a.keys < VEC || lds > (48 << 10)) {
            bias_grad_stream_kernel<T><<<grid, 1024, one, st>>>(a);
        } else {
            HPT_WITH_NC(d.nc, {
                constexpr int M = sizeof(T) == 4 ? (NC > 4 ? 4 : NC) : (NC > 2 ? 2 : NC);
                if (al) bias_grad_kernel<T, M, true><<<grid, d.threads, lds, st>>>(a);
                else bias_grad_kernel<T, M, false><<<grid, d.threads, lds, st>>>(a);
            });
        }
    });
    if (a.table_grad) launch_table(a, matrices, st);
}

}  // namespace hpt
