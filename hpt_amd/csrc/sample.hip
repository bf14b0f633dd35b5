// One token for each row of logits x, from a given number u in [0, 1).
//
// With the order of the row's tokens (larger logit first, equal ones by index) and weights w = exp((x - max) / temperature), every filter keeps a beginning of that
// order: the first top_k; of these the fewest whose weights reach top_p of theirs together; of these the ones with w >= min_p. So what is kept is
// a place of the order (key and index), and the token is the first, by index, at which the kept weights' sum is above u of their whole.
//
// Which token that is hangs on sums over the row: an error of 1e-7 of the sum, f32's, moves one of 10^5 borders across u in a row out of fifty. Weights and sums have 52
// bits here: with t = x log2 e 32 / temperature, w is 2^(floor(t) / 32) from a table of 32 times a polynomial in t - floor(t) (degree 5, 2e-15). f64 multiply-adds run
// at the rate of f32 ones, so the first launch still reads at some TB/s.
//
// Two launches. The first takes tiles of 8192 logits and leaves, by what the row's filters need: its threads' largest keys (top_k of at most 1024: only the first places
// matter); the sum of the weights (no filter); or the weights' sums by size, in buckets of an eighth of a power of two, as integers, whose sum has no order (with their
// numbers where top_k is larger). The second has a workgroup for each row: it finds the bucket in which a border lies, collects that bucket's logits, narrows the border to one
// place, and then looks through the one tile in which u's token lies.
#include <algorithm>

#include "top_rows.hpp"

namespace hpt {

namespace {

constexpr int kBuckets = 256, kCopies = 4;
constexpr int kFar = 32 * 128;             // weights below 2^-128 of the largest are 0

struct SampleHead {
    double top;     // 31 + 32 floor(t / 32) of the tile's largest: the octave that its weights are counted from
    double sum;     // of its weights, in that octave's units
    uint32_t most;  // the largest key
    uint32_t unused[3];
};
struct SampleBody {
    union {
        uint32_t keys[kTileGroups];
        struct {
            uint64_t mass[kBuckets];
            uint32_t count[kBuckets];
        };
    };
};

// ---- a row's settings -----------------------------------------------------------------------------

enum { BAD, FEW, PLAIN, SORTED };
__device__ __forceinline__ double number_of(const Setting& s, int64_t row) {
    if (!s.each) return s.all;
    if (s.dtype == HPT_F32) return ((const float*)s.each)[row];
    return s.dtype == HPT_I32 ? (double)((const int32_t*)s.each)[row] : (double)((const int64_t*)s.each)[row];
}
struct Settings {
    int mode, k;
    double steps, p, least;  // steps: of 1/32 octave for each unit of a logit
    __device__ __forceinline__ Settings(const SampleArgs& a, int64_t row) {
        double t = number_of(a.temperature, row);
        const double kk = number_of(a.top_k, row);
        p = number_of(a.top_p, row);
        least = number_of(a.min_p, row);
        k = kk >= 1.0 && kk < (double)a.cols ? (int)kk : a.cols;
        const bool bad = !(t == 0.0 || (t >= 1e-30 && t <= 1e30)) || p != p || least != least;
        if (t == 0.0) {  // the first of the order
            t = 1.0;
            k = 1;
        }
        if (p <= 0.0) k = 1;
        steps = 32.0 * 1.4426950408889634 / t;
        const bool few = k <= kMostTop && k < a.cols;
        mode = bad ? BAD : few || a.cols == 1 ? FEW : p >= 1.0 && least <= 0.0 && k == a.cols ? PLAIN : SORTED;
    }
};

// ---- weights --------------------------------------------------------------------------------------

// 2^(f / 32) for f in [0, 1): Taylor's polynomial at 1/2, written in powers of f.
struct Poly {
    double c[6];
};
constexpr Poly make_poly() {
    const double l = 0.6931471805599453 / 32.0;
    double a[6] = {};
    // e^(l / 2)
    double middle = 0.0, term = 1.0;
    for (int i = 0; i < 20; ++i) {
        middle += term;
        term *= (l / 2) / (i + 1);
    }
    a[0] = middle;
    for (int i = 1; i < 6; ++i) a[i] = a[i - 1] * l / i;
    Poly p{};
    for (int i = 0; i < 6; ++i) {
        double binomial = 1.0;
        for (int k = i; k >= 0; --k) {  // C(i, k) (-1/2)^(i - k)
            p.c[k] += a[i] * binomial;
            binomial = binomial * k / (i - k + 1) * -0.5;
        }
    }
    return p;
}
constexpr Poly kPoly = make_poly();

struct Weights {
    const double* table;  // 2^(j / 32) in LDS
    double steps, top;
    // How many steps below the top octave's end a logit lies (1000000: far, or -inf), and its weight's mantissa, in [1, 2).
    __device__ __forceinline__ int below(float x, double& f) const {
        const double t = (double)x * steps, n = floor(t);
        f = t - n;
        return (int)fmax(fmin(top - n, 1e6), 0.0);
    }
    __device__ __forceinline__ int below(float x) const {
        double f;
        return below(x, f);
    }
    __device__ __forceinline__ double mantissa(int r, double f) const {
        double v = kPoly.c[5];
#pragma unroll
        for (int i = 4; i >= 0; --i) v = fma(v, f, kPoly.c[i]);
        return v * table[31 - (r & 31)];
    }
    // In units of the top octave: in [1, 2) within it.
    __device__ __forceinline__ double of(float x) const {
        double f;
        const int r = below(x, f);
        return r < kFar ? ldexp(mantissa(r, f), -(r >> 5)) : 0.0;
    }
};
__device__ __forceinline__ double top_of(float most, double steps) { return 32.0 * floor((double)most * steps * (1.0 / 32.0)) + 31.0; }
__device__ __forceinline__ void make_table(double* table) {
    if (threadIdx.x < 32) table[threadIdx.x] = exp2(threadIdx.x * (1.0 / 32.0));
}
// Mantissas as integers, for sums without an order: of 2^-44 (in a larger vocabulary 2^-40), so that a row's are below 2^63. The same everywhere: equal weights
// reach a half of their sum at the half of their number.
struct Fixed {
    double base, unit;
    __device__ __forceinline__ explicit Fixed(int cols) : base(cols <= 1 << 18 ? 256.0 : 4096.0), unit(cols <= 1 << 18 ? 0x1p-44 : 0x1p-40) {}
    // 0 <= v < 2, rounded, from where it lies in the sum's mantissa
    __device__ __forceinline__ uint64_t operator()(double v) const { return __builtin_bit_cast(uint64_t, v + base) - __builtin_bit_cast(uint64_t, base); }
};
__device__ __forceinline__ double pow2(int n) { return ldexp(1.0, n); }
__device__ __forceinline__ bool no_number(uint32_t key, uint32_t inf, uint32_t neg) { return key >= inf || key <= neg; }

// ---- first launch ---------------------------------------------------------------------------------

template <class T>
__global__ __launch_bounds__(kTileGroups) void sample_tiles_kernel(const SampleArgs a, int64_t row0, int64_t rows) {
    constexpr int VEC = 16 / sizeof(T), V = kTileVecs<T>;
    __shared__ uint32_t tops[4];
    __shared__ double sums[4], table[32];
    __shared__ uint64_t mass[kBuckets * kCopies];
    __shared__ uint32_t count[kBuckets * kCopies];
    const Fixed fixed(a.cols);
    make_table(table);
    __syncthreads();
    for (int64_t at = blockIdx.x; at < rows * a.tiles; at += gridDim.x) {
        const int64_t row = quotient(at, a.tiles);
        const int tile = (int)(at - row * a.tiles);
        Pack<T, VEC> p[V];
        load_tile<T>((const T*)a.x + offset_of(a.kept, row0 + row), tile, a.cols, p);
        const Settings set(a, row0 + row);
        if (set.mode == BAD) continue;
        SampleBody& body = ((SampleBody*)a.bodies)[at];
        const uint32_t key = most_key<T>(p);
        if (set.mode == FEW) {
            ((KeyOf<T>*)body.keys)[threadIdx.x] = (KeyOf<T>)key;
            continue;
        }
        SampleHead& head = ((SampleHead*)a.heads)[at];
        const uint32_t most = block_reduce<MaxU>(key, tops);
        if (no_number(most, kInfKey<T>, kNegInfKey<T>)) {
            if (threadIdx.x == 0) {
                head.top = -__builtin_huge_val();
                head.sum = 0.0;
                head.most = most;
            }
            continue;
        }
        const Weights w{table, set.steps, top_of(value_of<T>(most), set.steps)};
        double sum = 0.0;
        if (set.mode == PLAIN) {
#pragma unroll
            for (int b = 0; b < V; ++b)
#pragma unroll
                for (int i = 0; i < VEC; ++i) sum += w.of(Elem<T>::widen(p[b].v[i]));
        } else {
            const bool counted = set.k < a.cols;
            for (int i = threadIdx.x; i < kBuckets * kCopies; i += kTileGroups) {
                mass[i] = 0;
                count[i] = 0;
            }
            __syncthreads();
            const int copy = threadIdx.x & (kCopies - 1);
#pragma unroll
            for (int b = 0; b < V; ++b)
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    double f;
                    const int r = w.below(Elem<T>::widen(p[b].v[i]), f);
                    const int bucket = min(r >> 2, kBuckets - 1);
                    // (the last bucket holds all that is below: in units of its own octave)
                    if (r < kFar) {
                        const double v = ldexp(w.mantissa(r, f), -max((r >> 5) - (kBuckets / 8 - 1), 0));
                        __hip_atomic_fetch_add(&mass[bucket * kCopies + copy], fixed(v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                        if (counted) __hip_atomic_fetch_add(&count[bucket * kCopies + copy], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                    }
                }
            __syncthreads();
            static_assert(kBuckets == kTileGroups, "a bucket a thread");
            uint64_t m = 0;
            uint32_t c = 0;
#pragma unroll
            for (int i = 0; i < kCopies; ++i) {
                m += mass[threadIdx.x * kCopies + i];
                c += count[threadIdx.x * kCopies + i];
            }
            body.mass[threadIdx.x] = m;
            if (counted) body.count[threadIdx.x] = c;
            sum = (double)m * fixed.unit * pow2(-(int)(threadIdx.x >> 3));
        }
        sum = block_reduce<SumD>(sum, sums);
        if (threadIdx.x == 0) {
            head.top = w.top;
            head.sum = sum;
            head.most = most;
        }
    }
}

// ---- second launch --------------------------------------------------------------------------------

struct SortedShared {
    uint64_t list[kMostList];
    uint64_t mass[kBuckets];  // of a digit
    uint32_t count[kBuckets];
    double row_mass[kBuckets];  // of a bucket of the row, in the top octave's units
    uint32_t row_count[kBuckets];
    uint64_t within[kMostParts];  // kept weights of a tile within the border's bucket
    uint16_t active[kMostParts];
    uint64_t few[64];
    uint32_t n, n_active;
    // what a search hands on
    int bucket;
    double before;          // weights, and number, of what is before the range
    uint32_t count_before;
    uint64_t lo, hi;
    uint64_t border;
    double reach;           // weights up to the border
};
struct PickShared {
    union {
        TopShared top;
        SortedShared sorted;
    };
    double part[kMostParts];  // kept weights of a tile
    int shift[kMostParts];    // by how many buckets its top octave is below the row's
    double table[32], place[16];
    uint32_t tops[16];
    double pick_before;
    int pick, pick_last;
    uint32_t token;
};

// A row as the second launch sees it.
template <class T> struct Row {
    const SampleArgs& a;
    const T* x;
    const SampleHead* heads;
    const SampleBody* bodies;
    Settings set;
    Weights w;
    Fixed fixed;
    uint32_t most;
    int index_bits;

    __device__ __forceinline__ uint64_t place(uint32_t key, uint32_t index) const { return ((uint64_t)key << index_bits) | ((1u << index_bits) - 1 - index); }
    __device__ __forceinline__ uint32_t key_at(uint64_t place) const { return (uint32_t)(place >> index_bits); }
    __device__ __forceinline__ uint32_t index_at(uint64_t place) const { return ((1u << index_bits) - 1) - ((uint32_t)place & ((1u << index_bits) - 1)); }
    __device__ __forceinline__ int bucket(uint32_t key) const { return min(w.below(value_of<T>(key)) >> 2, kBuckets - 1); }

    // The smallest key from `lo` to `most` of which `is` holds; it holds for `most`, and above any key of which it holds. Every wavefront for itself, 64 keys at a time.
    template <class Is> __device__ __forceinline__ uint32_t first_key(Is&& is) const {
        uint32_t lo = kNegInfKey<T> - 1, hi = most;  // not of lo, of hi
        while (hi - lo > 1) {
            const uint32_t step = (hi - lo + 63) / 64;
            const uint64_t at = (uint64_t)lo + (uint64_t)step * ((threadIdx.x & 63) + 1);
            const uint32_t key = at < hi ? (uint32_t)at : hi;
            const uint64_t yes = __ballot(key == hi || is(key));
            const int first = __builtin_ctzll(yes);
            const uint64_t top = (uint64_t)lo + (uint64_t)step * (first + 1);
            lo = lo + step * first;
            hi = top < hi ? (uint32_t)top : hi;
        }
        return hi;
    }
    // The largest key of a bucket that the row has something in.
    __device__ __forceinline__ uint32_t last_key(int b) const {
        return bucket(most) == b ? most : first_key([&](uint32_t key) { return bucket(key) < b; }) - 1;
    }
    // Calls f(on, place, value) of every logit of the tiles of s.active for whole wavefronts, in no order; `on`: there is one, and its place is in lo ... hi.
    template <class F> __device__ __forceinline__ void sweep(const SortedShared& s, uint64_t lo, uint64_t hi, F&& f) const {
        constexpr int VEC = 16 / sizeof(T), per = kTile / VEC;
        const uint32_t klo = key_at(lo), khi = key_at(hi);
        const int all = (int)s.n_active * per;
        for (int i0 = 0; i0 < all; i0 += blockDim.x) {
            const int i = i0 + threadIdx.x;
            Pack<T, VEC> p;
            int e = a.cols;
            if (i < all) {
                const int v = s.active[i / per] * per + i % per;
                if (v * VEC < a.cols) {
                    e = v * VEC;
                    p = logit_vec<T>(x, v, a.cols);
                }
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const uint32_t key = e + j < a.cols ? key_of(p.v[j]) : 0;
                bool on = key >= klo && key <= khi && e + j < a.cols;
                const uint64_t at = place(key, on ? e + j : 0);
                on = on && at >= lo && at <= hi;
                f(on, at, p.v[j]);
            }
        }
    }
};

// The tiles that have logits in a bucket of the row.
template <class T> __device__ __forceinline__ void find_active(const Row<T>& r, PickShared& s, int bucket) {
    SortedShared& q = s.sorted;
    __syncthreads();
    if (threadIdx.x == 0) q.n_active = 0;
    __syncthreads();
    for (int t = threadIdx.x; t < r.a.tiles; t += blockDim.x) {
        const int src = bucket - s.shift[t];
        // (of the last bucket anything may be there, also what weighs nothing)
        const bool on = bucket == kBuckets - 1 || (src >= 0 && r.bodies[t].mass[src] != 0);
        if (on) q.active[atomicAdd(&q.n_active, 1u)] = (uint16_t)t;
    }
    __syncthreads();
}

// The border: the first place of the order at which the number of tokens reaches `k` (BY_COUNT) or their weights reach `target`. Returns the place (0: all of the row
// is before it), in s.sorted.reach the weights up to it. `listed`: the bucket whose logits s.sorted.list holds, all of them, q.n in number.
template <bool BY_COUNT, class T> __device__ __forceinline__ uint64_t find_border(const Row<T>& r, PickShared& s, uint32_t k, double target, int& listed) {
    SortedShared& q = s.sorted;
    __syncthreads();
    if (threadIdx.x < 64) {
        const int lane = threadIdx.x;
        double m[4], sum = 0.0;
        uint32_t c[4], number = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            m[i] = q.row_mass[lane * 4 + i];
            c[i] = BY_COUNT ? q.row_count[lane * 4 + i] : 0;
            sum += m[i];
            number += c[i];
        }
        double upto = sum;
        uint32_t number_upto = number;
#pragma unroll
        for (int w = 1; w < 64; w <<= 1) {
            union { double d; int i[2]; } in, out;
            in.d = upto;
            out.i[0] = __shfl_up(in.i[0], w, 64);
            out.i[1] = __shfl_up(in.i[1], w, 64);
            const uint32_t o = __shfl_up(number_upto, w, 64);
            if (lane >= w) {
                upto += out.d;
                number_upto += o;
            }
        }
        double before = upto - sum;
        uint32_t number_before = number_upto - number;
        // (the difference may be a rounding off the sum before: the lane before's own)
        {
            union { double d; int i[2]; } in, out;
            in.d = upto;
            out.i[0] = __shfl_up(in.i[0], 1, 64);
            out.i[1] = __shfl_up(in.i[1], 1, 64);
            before = lane ? out.d : 0.0;
        }
        const uint64_t reach = __ballot(BY_COUNT ? number_upto >= k : upto >= target);
        const uint64_t some = __ballot(BY_COUNT ? number > 0 : sum > 0.0);
        const int at = reach ? __builtin_ctzll(reach) : 63 - __builtin_clzll(some | 1);
        if (lane == at) {
            int b = 0;
            // (where rounding keeps the sum below the target, the last bucket with anything)
            int last = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (BY_COUNT ? c[i] > 0 : m[i] > 0.0) last = i;
            bool found = false;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (!found && i <= last) {
                    const bool here = i == last || (BY_COUNT ? number_before + c[i] >= k : before + m[i] >= target);
                    if (here) {
                        found = true;
                        b = i;
                    } else {
                        before += m[i];
                        number_before += c[i];
                    }
                }
            q.bucket = lane * 4 + b;
            q.before = before;
            q.count_before = number_before;
        }
    }
    __syncthreads();
    const int bucket = q.bucket;
    double before = q.before;
    uint32_t count_before = q.count_before;
    const uint32_t klo = bucket == kBuckets - 1 ? kNegInfKey<T> : r.first_key([&](uint32_t key) { return r.bucket(key) <= bucket; });
    const uint32_t khi = r.last_key(bucket);
    uint64_t lo = r.place(klo, (1u << r.index_bits) - 1), hi = r.place(khi, 0);
    const double unit = pow2(-(bucket >> 3)) * r.fixed.unit;  // of the bucket's octave
    auto weight = [&](float x) { return r.fixed(r.w.of(x) * pow2(bucket >> 3)); };
    bool have = listed == bucket;
    uint32_t n = have ? q.n : 0xFFFFFFFFu;
    if (!have) {
        find_active(r, s, bucket);
        listed = -1;
    }
    bool first = true;
    while (true) {
        if (!have && (first || n <= kMostList)) {
            __syncthreads();
            if (threadIdx.x == 0) q.n = 0;
            __syncthreads();
            r.sweep(q, lo, hi, [&](bool on, uint64_t at, T) {
                if (__any(on)) {
                    const uint32_t i = reserve(on, &q.n);
                    if (on && i < kMostList) q.list[i] = at;
                }
            });
            __syncthreads();
            n = q.n;
            have = n <= kMostList;
            if (have && first) listed = bucket;
            if (n == 0) return 0;
        }
        first = false;
        if (have && n <= 64) break;
        // by eight bits of the place
        __syncthreads();
        for (int i = threadIdx.x; i < kBuckets; i += blockDim.x) {
            q.mass[i] = 0;
            q.count[i] = 0;
        }
        __syncthreads();
        const uint64_t width = hi - lo;
        const int bits = width ? 64 - __builtin_clzll(width) : 0, shift = bits > 8 ? bits - 8 : 0;
        auto count = [&](uint64_t at, float x) {
            const int d = (int)((at - lo) >> shift);
            __hip_atomic_fetch_add(&q.count[d], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            __hip_atomic_fetch_add(&q.mass[d], weight(x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        };
        if (have) {
            const uint32_t all = min(q.n, (uint32_t)kMostList);
            for (uint32_t i = threadIdx.x; i < all; i += blockDim.x) {
                const uint64_t at = q.list[i];
                if (at >= lo && at <= hi) count(at, value_of<T>(r.key_at(at)));
            }
        } else {
            r.sweep(q, lo, hi, [&](bool on, uint64_t at, T v) {
                if (on) count(at, Elem<T>::widen(v));
            });
        }
        __syncthreads();
        if (threadIdx.x < 64) {
            const int lane = threadIdx.x;
            uint64_t m[4], sum = 0;
            uint32_t c[4], number = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                m[i] = q.mass[255 - (lane * 4 + i)];
                c[i] = q.count[255 - (lane * 4 + i)];
                sum += m[i];
                number += c[i];
            }
            uint64_t upto = sum;
            uint32_t number_upto = number;
#pragma unroll
            for (int w = 1; w < 64; w <<= 1) {
                const uint32_t o0 = __shfl_up((uint32_t)upto, w, 64), o1 = __shfl_up((uint32_t)(upto >> 32), w, 64), o = __shfl_up(number_upto, w, 64);
                if (lane >= w) {
                    upto += (uint64_t)o1 << 32 | o0;
                    number_upto += o;
                }
            }
            auto reached = [&](uint64_t m, uint32_t c) { return BY_COUNT ? count_before + c >= k : before + (double)m * unit >= target; };
            const uint64_t reach = __ballot(number > 0 && reached(upto, number_upto));
            const uint64_t some = __ballot(number > 0);
            const int at = reach ? __builtin_ctzll(reach) : 63 - __builtin_clzll(some | 1);
            if (lane == at) {
                uint64_t above = upto - sum;
                uint32_t number_above = number_upto - number;
                int last = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (c[i] > 0) last = i;
                int d = 0;
                bool found = false;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (!found && i <= last) {
                        if (i == last || (c[i] > 0 && reached(above + m[i], number_above + c[i]))) {
                            found = true;
                            d = i;
                        } else {
                            above += m[i];
                            number_above += c[i];
                        }
                    }
                const uint64_t digit = 255 - (lane * 4 + d);
                q.lo = lo + (digit << shift);
                q.hi = min(hi, q.lo + ((1ull << shift) - 1));
                q.before = before + (double)above * unit;
                q.count_before = count_before + number_above;
                q.few[0] = q.count[digit];
            }
        }
        __syncthreads();
        lo = q.lo;
        hi = q.hi;
        before = q.before;
        count_before = q.count_before;
        n = (uint32_t)q.few[0];
        __syncthreads();
    }
    // at most 64 are left: a lane each
    __syncthreads();
    if (threadIdx.x == 0) q.n_active = 0;  // (their number; the tiles are not needed any more)
    __syncthreads();
    {
        const uint32_t all = q.n;
        for (uint32_t i0 = 0; i0 < all; i0 += blockDim.x) {
            const uint32_t i = i0 + threadIdx.x;
            const uint64_t at = i < all ? q.list[i] : 0;
            const bool on = i < all && at >= lo && at <= hi;
            if (__any(on)) {
                const uint32_t to = reserve(on, &q.n_active);
                if (on && to < 64) q.few[to] = at;
            }
        }
    }
    __syncthreads();
    if (threadIdx.x < 64) {
        const int lane = threadIdx.x;
        const int left = (int)q.n_active;
        const uint64_t mine = lane < left ? q.few[lane] : 0;
        const uint64_t m = lane < left ? weight(value_of<T>(r.key_at(mine))) : 0;
        uint64_t upto = 0;
        uint32_t number = 0;
        for (int j = 0; j < left; ++j) {
            const uint64_t other = q.few[j];
            const uint64_t om = (uint64_t)(uint32_t)__shfl((uint32_t)(m >> 32), j, 64) << 32 | (uint32_t)__shfl((uint32_t)m, j, 64);
            if (other >= mine) {
                upto += om;
                ++number;
            }
        }
        const bool reached = lane < left && (BY_COUNT ? count_before + number >= k : before + (double)upto * unit >= target);
        // the first that reaches it, or the last there is
        const uint32_t score = reached ? 1024 - number : lane < left ? number : 0;
        if (score == group_reduce<MaxU>(score, 64)) {
            q.border = mine;
            q.reach = before + (double)upto * unit;
        }
    }
    __syncthreads();
    return q.border;
}

// Writes a row's answer.
template <class T> __device__ __forceinline__ void answer(const SampleArgs& a, int64_t row, int64_t token, double logp) {
    if (a.token64) ((int64_t*)a.token)[row] = token;
    else ((int32_t*)a.token)[row] = (int32_t)token;
    a.logp[row] = (float)logp;
}

template <class T>
__global__ __launch_bounds__(1024) void sample_pick_kernel(const SampleArgs a, int64_t row0, int64_t rows) {
    constexpr int VEC = 16 / sizeof(T);
    __shared__ PickShared s;
    make_table(s.table);
    for (int64_t at = blockIdx.x; at < rows; at += gridDim.x) {
        const int64_t row = row0 + at;
        __syncthreads();
        Row<T> r{a, (const T*)a.x + offset_of(a.kept, row), (const SampleHead*)a.heads + at * a.tiles, (const SampleBody*)a.bodies + at * a.tiles,
                 Settings(a, row), Weights{s.table, 0.0, 0.0}, Fixed(a.cols), 0, a.cols > 1 ? 32 - __builtin_clz((unsigned)a.cols - 1) : 0};
        const Settings& set = r.set;
        r.w.steps = set.steps;
        double u = a.u[row];
        u = u > 0.0 ? u : 0.0;
        if (set.mode == BAD) {
            if (threadIdx.x == 0) answer<T>(a, row, -1, __builtin_nan(""));
            continue;
        }
        if (set.mode == FEW) {
            // (the tiles' keys lie a body apart, one tile's side by side)
            const int k = set.k;
            const int n = collect_top<T>(s.top, r.x, a.cols, (const KeyOf<T>*)r.bodies, a.tiles, k, sizeof(SampleBody));
            uint64_t* order = (uint64_t*)s.top.groups;
            static_assert(sizeof s.top.groups >= kMostTop * sizeof(uint64_t), "");
            rank_top(s.top, n, k, [&](int rank, uint64_t p) { order[rank] = p; });
            __syncthreads();
            const uint32_t most = key_of_place(order[0]);
            if (no_number(most, kInfKey<T>, kNegInfKey<T>)) {
                if (threadIdx.x == 0) answer<T>(a, row, -1, __builtin_nan(""));
                continue;
            }
            r.w.top = top_of(value_of<T>(most), set.steps);
            double* weight = (double*)s.top.list;
            static_assert(sizeof s.top.list >= kMostTop * sizeof(double), "");
            const int each = (k + (int)blockDim.x - 1) / (int)blockDim.x, i0 = min((int)threadIdx.x * each, k), i1 = min(i0 + each, k);
            double mine = 0.0;
            for (int i = i0; i < i1; ++i) mine += weight[i] = r.w.of(value_of<T>(key_of_place(order[i])));
            double all;
            const double before = scan_before(mine, s.place, all);
            // how many are kept
            if (threadIdx.x == 0) s.pick = k;
            __syncthreads();
            const double target = set.p * all, least = fmin(set.least, 1.0) * weight[0];
            double upto = before;
            int cut = k;
            for (int i = i0; i < i1 && cut == k; ++i) {
                if (weight[i] < least && i > 0) cut = i;
                upto += weight[i];
                if (set.p < 1.0 && upto >= target) cut = min(cut, i + 1);
            }
            if (cut < k) atomicMin(&s.pick, cut);
            __syncthreads();
            const int kept = s.pick;
            upto = before;
            for (int i = i0; i < i1; ++i) {
                upto += weight[i];
                if (i == kept - 1) s.pick_before = upto;
            }
            if (threadIdx.x == 0) s.token = 0;
            __syncthreads();
            // u's token: the last by index whose weights before it do not exceed u's part
            const double part = u * s.pick_before;
            for (int i = threadIdx.x; i < kept; i += blockDim.x) {
                const uint32_t index = index_of(order[i]);
                double sum = 0.0;
#pragma unroll 4
                for (int j = 0; j < kept; ++j) sum += index_of(order[j]) < index ? weight[j] : 0.0;
                if (weight[i] > 0.0 && sum <= part) atomicMax(&s.token, index + 1);
            }
            __syncthreads();
            for (int i = threadIdx.x; i < kept; i += blockDim.x)
                if (index_of(order[i]) + 1 == s.token) answer<T>(a, row, s.token - 1, log(weight[i] / s.pick_before));
            continue;
        }
        // the tiles together
        double top = -__builtin_huge_val();
        uint32_t most = 0;
        for (int t = threadIdx.x; t < a.tiles; t += blockDim.x) {
            top = fmax(top, r.heads[t].top);
            most = max(most, r.heads[t].most);
        }
        most = block_reduce<MaxU>(most, s.tops);
        struct MaxD {
            __device__ static __forceinline__ double comb(double a, double b) { return fmax(a, b); }
        };
        top = block_reduce<MaxD>(top, s.place);
        if (no_number(most, kInfKey<T>, kNegInfKey<T>)) {
            if (threadIdx.x == 0) answer<T>(a, row, -1, __builtin_nan(""));
            continue;
        }
        r.most = most;
        r.w.top = top;
        double all = 0.0;
        for (int t = threadIdx.x; t < a.tiles; t += blockDim.x) {
            const int shift = (int)fmin((top - r.heads[t].top) * 0.25, 1e6);
            s.shift[t] = shift;
            s.part[t] = shift < 8 * 1024 ? ldexp(r.heads[t].sum, -(shift >> 3)) : 0.0;
            all += s.part[t];
        }
        uint64_t border = 0;
        if (set.mode == SORTED) {
            SortedShared& q = s.sorted;
            const bool counted = set.k < a.cols;
            all = block_reduce<SumD>(all, s.place);
            __syncthreads();
            // the row's buckets
            double mine = 0.0;
            uint32_t number = 0;
            if ((int)threadIdx.x < kBuckets - 1) {
                const int b = threadIdx.x;
                for (int t = 0; t < a.tiles; ++t) {
                    const int src = b - s.shift[t];
                    if (src < 0) continue;
                    mine += (double)r.bodies[t].mass[src];
                    if (counted) number += r.bodies[t].count[src];
                }
                mine *= pow2(-(b >> 3)) * r.fixed.unit;
                q.row_mass[b] = mine;
                q.row_count[b] = number;
            }
            const double upper = block_reduce<SumD>(mine, s.place);
            struct SumU {
                __device__ static __forceinline__ uint32_t comb(uint32_t a, uint32_t b) { return a + b; }
            };
            number = block_reduce<SumU>(number, s.tops);
            if (threadIdx.x == 0) {
                q.row_mass[kBuckets - 1] = fmax(all - upper, 0.0);
                q.row_count[kBuckets - 1] = a.cols - number;
            }
            int listed = -1;
            double whole = all;
            if (counted) {
                border = find_border<true>(r, s, set.k, 0.0, listed);
                whole = q.reach;
            }
            if (set.p < 1.0) border = max(border, find_border<false>(r, s, 0, set.p * whole, listed));
            if (set.least > 0.0) {
                const double least = fmin(set.least, 1.0) * r.w.of(value_of<T>(most));
                border = max(border, (uint64_t)r.first_key([&](uint32_t key) { return r.w.of(value_of<T>(key)) >= least; }) << r.index_bits);
            }
            __syncthreads();
            if (border) {
                // what is kept of each tile: its buckets above the border's, and within that bucket the logits up to the border
                const int bucket = r.bucket(r.key_at(border));
                for (int t = threadIdx.x; t < a.tiles; t += blockDim.x) q.within[t] = 0;
                if (listed != bucket) find_active(r, s, bucket);
                __syncthreads();
                const double up = pow2(bucket >> 3);
                auto add = [&](uint64_t at, float x) {
                    __hip_atomic_fetch_add(&q.within[r.index_at(at) / kTile], r.fixed(r.w.of(x) * up), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                };
                if (listed == bucket) {
                    for (uint32_t i = threadIdx.x; i < q.n; i += blockDim.x) {
                        const uint64_t p = q.list[i];
                        if (p >= border) add(p, value_of<T>(r.key_at(p)));
                    }
                } else {
                    r.sweep(q, border, r.place(r.last_key(bucket), 0), [&](bool on, uint64_t p, T v) {
                        if (on) add(p, Elem<T>::widen(v));
                    });
                }
                __syncthreads();
                for (int t = threadIdx.x >> 6; t < a.tiles; t += blockDim.x >> 6) {
                    double kept = 0.0;
#pragma unroll
                    for (int i = 0; i < kBuckets / 64; ++i) {
                        const int b = (threadIdx.x & 63) + 64 * i, src = b - s.shift[t];
                        if (b < bucket && src >= 0) kept += (double)r.bodies[t].mass[src] * pow2(-(b >> 3));
                    }
                    kept = group_reduce<SumD>(kept, 64) * r.fixed.unit;
                    if ((threadIdx.x & 63) == 0) s.part[t] = kept + (double)q.within[t] * (pow2(-(bucket >> 3)) * r.fixed.unit);
                }
            }
        }
        __syncthreads();
        // u's tile: the first at which the sum exceeds u of the whole
        const int each = (a.tiles + (int)blockDim.x - 1) / (int)blockDim.x, t0 = min((int)threadIdx.x * each, a.tiles), t1 = min(t0 + each, a.tiles);
        double mine = 0.0;
        for (int t = t0; t < t1; ++t) mine += s.part[t];
        double whole;
        double before = scan_before(mine, s.place, whole);
        if (threadIdx.x == 0) {
            s.pick = INT32_MAX;
            s.pick_last = 0;
        }
        __syncthreads();
        const double target = u * whole;
        double upto = before;
        for (int t = t0; t < t1; ++t) {
            if (s.part[t] > 0.0) atomicMax(&s.pick_last, t);
            upto += s.part[t];
            if (s.part[t] > 0.0 && upto > target) {
                atomicMin(&s.pick, t);
                break;
            }
        }
        __syncthreads();
        const int tile = s.pick == INT32_MAX ? s.pick_last : s.pick;
        if (t0 <= tile && tile < t1) {
            for (int t = t0; t < tile; ++t) before += s.part[t];
            s.pick_before = before;
        }
        __syncthreads();
        const double rest = target - s.pick_before;
        // and its token there
        const int run = kTile / (int)blockDim.x, e0 = tile * kTile + (int)threadIdx.x * run;
        auto look = [&](auto&& f) {
            for (int v = 0; v < run / VEC; ++v) {
                const int e = e0 + v * VEC;
                if (e >= a.cols) break;
                const Pack<T, VEC> p = logit_vec<T>(r.x, e / VEC, a.cols);
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    if (e + i < a.cols && r.place(key_of(p.v[i]), e + i) >= border) f(e + i, r.w.of(Elem<T>::widen(p.v[i])));
            }
        };
        mine = 0.0;
        look([&](int, double w) { mine += w; });
        double tile_sum;
        const double here = scan_before(mine, s.place, tile_sum);
        if (threadIdx.x == 0) {
            s.pick = INT32_MAX;
            s.pick_last = -1;
        }
        __syncthreads();
        if (mine > 0.0) {
            double sum = here;
            int last = -1, first = INT32_MAX;
            look([&](int e, double w) {
                if (w > 0.0) {
                    last = e;
                    sum += w;
                    if (sum > rest && e < first) first = e;
                }
            });
            atomicMax(&s.pick_last, last);
            if (first != INT32_MAX) atomicMin(&s.pick, first);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            const int token = s.pick == INT32_MAX ? s.pick_last : s.pick;
            answer<T>(a, row, token, token < 0 ? __builtin_nan("") : log(fmin(r.w.of(Elem<T>::widen(r.x[token])) / whole, 1.0)));
        }
    }
}

}  // namespace

size_t sample_row_bytes(int64_t cols) { return (size_t)((cols + kTile - 1) / kTile) * (sizeof(SampleHead) + sizeof(SampleBody)); }

void launch_sample(int dtype, const SampleArgs& args, hipStream_t st) {
    SampleArgs a = args;
    static_assert(sizeof(SampleHead) % 16 == 0 && sizeof(SampleBody) % 16 == 0, "both arrays are aligned");
    a.bodies = (char*)a.heads + (size_t)a.run * a.tiles * sizeof(SampleHead);
    HPT_WITH_TYPE(dtype, {
        for (int64_t row0 = 0; row0 < a.rows; row0 += a.run) {
            const int64_t rows = std::min(a.run, a.rows - row0);
            sample_tiles_kernel<T><<<(unsigned)std::min<int64_t>(rows * a.tiles, 1 << 20), kTileGroups, 0, st>>>(a, row0, rows);
            sample_pick_kernel<T><<<(unsigned)std::min<int64_t>(rows, 1 << 20), rows <= 512 ? 1024 : 256, 0, st>>>(a, row0, rows);
        }
    });
}

}  // namespace hpt
