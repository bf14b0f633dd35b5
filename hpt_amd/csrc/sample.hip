// One token for each row of logits x, from a given number u in [0, 1).
//
// With the order of the row's tokens (larger logit first, equal ones by index) and weights w = exp((x - max) / temperature), every filter keeps a beginning of that
// order: the first top_k; of these the fewest whose weights reach top_p of theirs together; of these the ones with w >= min_p. So what is kept is
// a place of the order (key and index), and the token is the first, by index, at which the kept weights' sum is above u of their whole.
//
// Which token that is hangs on sums over the row: an error of 1e-7 of the sum, f32's, moves one of 10^5 borders across u in a row out of fifty. Weights and sums are of 64
// bits here: with t = x log2 e 128 / temperature and n the whole number next to it, w is 2^(n / 128), from a table of 128, times a polynomial in t - n (degree 3, 3e-13), and whole
// numbers of a bucket are of 2^-44 or 2^-40 of an octave: what is decided is the definition's wherever no border lies within 2^-36 of the row's sum of it. f64 multiply-adds run at the rate of f32 ones, so the first launch still reads at some TB/s; it is bound by its instructions, 16 for each logit.
//
// Two launches. The first takes tiles of 8192 logits and leaves, by what the row's filters need: the largest keys of its groups (top_k of at most 1024: only the first places
// matter); the sum of the weights (no filter); or the weights' sums by size, in buckets of an eighth of a power of two, as integers, whose sum has no order (with their
// numbers where top_k is larger). The second has a workgroup for each row: it finds the bucket in which a border lies, collects that bucket's logits, narrows the border to one
// place, and then looks through the one tile in which u's token lies. (Very many rows of which at most 64 places matter take a wavefront each.)
//
// us of the two launches, bf16 [2048, 50257] (206 MB): without a filter 85 + 14 (2.4 TB/s in the first), top_k 50 39 + 24 (5.3), 600 39 + 99, top_p 0.9 137 + 108 (1.5: two LDS additions' worth of
// instructions more). bf16 [1, 152000] with top_k 20 and top_p 0.8 2.5 + 10.5, f32 [33, 50257] with top_p 0.95 8 + 27, [64, 152000] with settings for each row 14 + 43: the steps of one workgroup, most of
// them the collection of a bucket, at a compute unit's own rate.
#include <algorithm>

#include "top_rows.hpp"

namespace hpt {

namespace {

constexpr int kSteps = 128;                  // of a power of two
constexpr int kBuckets = 256, kCopies = 8;   // of an eighth of a power of two
constexpr int kBucketSteps = kSteps / 8;
constexpr int kFar = kSteps * 128;           // weights below 2^-128 of the largest are 0

// What a tile leaves (of each of its wavefronts' 2048 logits, where there is no filter).
struct SampleHead {
    double sum;     // of the weights, in units of the octave of the largest
    uint32_t most;  // the largest key
    uint32_t unused;
};
struct SampleTile {
    SampleHead heads[kTileWaves];
    union {
        uint32_t keys[kTileGroups];
        struct {
            double mass[kBuckets];     // of a bucket and all above it, in units of the tile's top octave
            uint32_t count[kBuckets];  // likewise
        };
    };
};

// ---- a row's settings -----------------------------------------------------------------------------

enum Mode { BAD, FEW, PLAIN, SORTED, ANY };
__device__ __forceinline__ double number_of(const Setting& s, int64_t row) {
    if (!s.each) return s.all;
    if (s.dtype == HPT_F32) return ((const float*)s.each)[row];
    return s.dtype == HPT_I32 ? (double)((const int32_t*)s.each)[row] : (double)((const int64_t*)s.each)[row];
}
struct Settings {
    int mode, k;
    double steps, p, least;  // steps: of each unit of a logit
    // (the host, too: settings for all rows have kernels of their own)
    __host__ __device__ __forceinline__ Settings(double t, double kk, double p, double least, int cols) : p(p), least(least) {
        k = kk >= 1.0 && kk < (double)cols ? (int)kk : cols;
        const bool bad = !(t == 0.0 || (t >= 1e-30 && t <= 1e30)) || p != p || least != least;
        if (t == 0.0) {  // the first of the order
            t = 1.0;
            k = 1;
        }
        if (p <= 0.0) k = 1;
        steps = kSteps * 1.4426950408889634 / t;
        const bool few = k <= kMostTop && k < cols;
        mode = bad ? BAD : few || cols == 1 ? FEW : p >= 1.0 && least <= 0.0 && k == cols ? PLAIN : SORTED;
    }
    // of a row; `all`: those for all rows
    template <int MODE> static __device__ __forceinline__ Settings of(const SampleArgs& a, const Settings& all, int64_t row) {
        if constexpr (MODE == ANY) return Settings(a, row);
        else return all;
    }
    __device__ __forceinline__ Settings(const SampleArgs& a, int64_t row)
        : Settings(number_of(a.temperature, row), number_of(a.top_k, row), number_of(a.top_p, row), number_of(a.min_p, row), a.cols) {}
};

// ---- weights --------------------------------------------------------------------------------------

// 2^(f / 128) for |f| <= 1/2 (Taylor's polynomial, its next term by the quadratic next to it on that range), and 2^(j / 128).
struct Powers {
    double c[4], table[kSteps];
};
constexpr Powers make_powers() {
    const double l = 0.6931471805599453 / kSteps, next = l * l * l * l / 24;
    Powers p{};
    p.c[0] = 1.0 - next / 128;
    p.c[1] = l;
    p.c[2] = l * l / 2 + next / 4;
    p.c[3] = l * l * l / 6;
    for (int j = 0; j < kSteps; ++j) {
        double sum = 0.0, term = 1.0;
        for (int i = 1; i < 30; ++i) {
            sum += term;
            term *= l * j / i;
        }
        p.table[j] = sum;
    }
    return p;
}
__device__ constexpr Powers kPowers = make_powers();

// Whole numbers next to t, in the low bits of a sum (|t| < 2^51).
constexpr double kRound = 6755399441055744.0;  // 1.5 2^52
struct Weights {
    const double* table;  // 2^(j / 128) in LDS
    double steps;
    double round;  // kRound less the whole number that the largest's octave begins with, a multiple of 128: sums with it have steps above that in their low bits
    // `most`: the largest logit, a number. Where t would leave the whole numbers' range the steps are shortened: there, logits that differ do so by octaves beyond counting.
    __device__ __forceinline__ Weights(const double* table, float most, double steps) : table(table), steps(steps) {
        if (fabs((double)most * steps) > 0x1p49) this->steps = 0x1p49 / fabs((double)most);
        round = kRound - floor((fma((double)most, this->steps, kRound) - kRound) / kSteps) * kSteps;
    }
    // Steps above the beginning of the largest's octave: 0 to 127 within it, negative below.
    __device__ __forceinline__ int above(float x) const { return (int)(uint32_t)__builtin_bit_cast(uint64_t, fma((double)x, steps, round)); }
    // Likewise of a logit that is not below `lowest`, and its weight's mantissa, in [1, 2) or next to it.
    __device__ __forceinline__ int above(double x, double& mantissa) const {
        const double sum = fma(x, steps, round), f = fma(x, steps, round - sum);  // (exact but for one rounding, whatever t's size)
        const int n = (int)(uint32_t)__builtin_bit_cast(uint64_t, sum);
        double v = kPowers.c[3];
#pragma unroll
        for (int i = 2; i >= 0; --i) v = fma(v, f, kPowers.c[i]);
        mantissa = v * table[n & (kSteps - 1)];
        return n;
    }
    // The lowest logit that `above` may be asked for: 96 octaves down weigh nothing. (64 bits tell it from the largest, whose t is below 2^50.)
    __device__ __forceinline__ double lowest(float most) const { return (double)most - 96.0 * kSteps / steps; }

    // Of any logit: how many steps below the top octave's end (kFar: at least so many), and its weight in units of the top octave.
    __device__ __forceinline__ int below_any(float x, float most) const {
        const bool far = ((double)most - (double)x) * steps >= 100.0 * kSteps;
        return far ? kFar : kSteps - 1 - above(x);
    }
    __device__ __forceinline__ double of(float x, float most) const {
        const bool far = ((double)most - (double)x) * steps >= 100.0 * kSteps;
        double v;
        const int n = above(far ? most : x, v);
        return far ? 0.0 : moved(v, n);
    }
    // v 2^(n / 128), rounded down to whole octaves (of a number v that is not small), by its exponent
    static __device__ __forceinline__ double moved(double v, int n) {
        static_assert(kSteps == 1 << 7, "an octave is 2^20 of the upper word");
        return __hiloint2double((int)((uint32_t)__double2hiint(v) + ((uint32_t)(n & ~(kSteps - 1)) << (20 - 7))), __double2loint(v));
    }
};
__device__ __forceinline__ void make_table(double* table) {
    if (threadIdx.x < kSteps) table[threadIdx.x] = kPowers.table[threadIdx.x];
}
// Mantissas as integers, for sums without an order: of 2^-44 (in a larger vocabulary 2^-40), so that a row's are below 2^63. The same everywhere: equal weights
// reach a half of their sum at the half of their number.
struct Fixed {
    double base, unit;
    uint32_t upper;  // of the base's words: the other is 0
    __device__ __forceinline__ explicit Fixed(int cols) : base(cols <= 1 << 18 ? 256.0 : 4096.0), unit(cols <= 1 << 18 ? 0x1p-44 : 0x1p-40), upper(cols <= 1 << 18 ? 0x40700000u : 0x40B00000u) {}
    // 0 <= v < 2, rounded, from where it lies in the sum's mantissa
    __device__ __forceinline__ uint64_t operator()(double v) const {
        const double sum = v + base;
        return (uint64_t)((uint32_t)__double2hiint(sum) - upper) << 32 | (uint32_t)__double2loint(sum);
    }
};
__device__ __forceinline__ double pow2(int n) { return __builtin_bit_cast(double, (uint64_t)(1023 + n) << 52); }  // |n| < 1000
template <class T> __device__ __forceinline__ bool no_number(uint32_t key) { return key >= kInfKey<T> || key <= kNegInfKey<T>; }

// ---- first launch ---------------------------------------------------------------------------------

template <class T, int MODE>
__global__ __launch_bounds__(kTileGroups) void sample_tiles_kernel(const SampleArgs a, const Settings all, int64_t row0) {
    constexpr int VEC = 16 / sizeof(T), V = kTileVecs<T>;
    constexpr bool BUCKETS = MODE == SORTED || MODE == ANY;
    __shared__ uint32_t tops[4];
    __shared__ double sums[4], table[MODE == FEW ? 1 : kSteps];
    __shared__ uint64_t mass[BUCKETS ? kBuckets * kCopies : 1];
    __shared__ uint32_t count[BUCKETS ? kBuckets * kCopies : 1], counts[4];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t row = blockIdx.y;
    const Settings set = Settings::of<MODE>(a, all, row0 + row);
    const int mode = MODE == ANY ? set.mode : MODE;
    if (mode == BAD) return;
    const LogitRow<T> x((const T*)a.x + offset_of(a.kept, row0 + row), a.cols);
    if (mode != FEW) {
        make_table(table);
        __syncthreads();
    }
    for (int at = blockIdx.x; at < a.tiles; at += gridDim.x) {
        SampleTile& tile = ((SampleTile*)a.tiles_scratch)[row * a.tiles + at];
        Pack<T, VEC> p[V];
        load_tile<T>(x, at, p);
        if (mode == FEW) {
            ((KeyOf<T>*)tile.keys)[threadIdx.x] = (KeyOf<T>)group_key<T>(p);
            continue;
        }
        uint32_t key = 0;
#pragma unroll
        for (int b = 0; b < V; ++b) key = max(key, most_key<T>(p[b]));
        key = wave_max(key);
        double sum = 0.0;
        if (!BUCKETS || mode == PLAIN) {
            // a wavefront's part, in the octave of its own largest: nobody waits for anybody
            if (!no_number<T>(key)) {
                const float most = value_of<T>(key);
                const Weights w(table, most, set.steps);
                const double lowest = w.lowest(most);
#pragma unroll
                for (int b = 0; b < V; ++b)
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        double v;
                        const int n = w.above(fmax((double)Elem<T>::widen(p[b].v[i]), lowest), v);
                        sum += Weights::moved(v, n);
                    }
                sum = group_reduce<SumD>(sum, 64);
            }
            if (lane == 0) {
                tile.heads[wave].sum = sum;
                tile.heads[wave].most = key;
            }
            continue;
        }
        if constexpr (BUCKETS) {
            __syncthreads();
            if (lane == 0) tops[wave] = key;
            for (int i = threadIdx.x; i < kBuckets * kCopies; i += kTileGroups) {
                mass[i] = 0;
                count[i] = 0;
            }
            __syncthreads();
            key = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
            if (!no_number<T>(key)) {
                const bool counted = set.k < a.cols;
                const float most = value_of<T>(key);
                const Weights w(table, most, set.steps);
                const Fixed fixed(a.cols);
                const double lowest = w.lowest(most);
                const int copy = threadIdx.x & (kCopies - 1);
#pragma unroll
                for (int b = 0; b < V; ++b)
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        double v;
                        const int n = w.above(fmax((double)Elem<T>::widen(p[b].v[i]), lowest), v);
                        const uint32_t bucket = min((uint32_t)(kSteps - 1 - n) / kBucketSteps, (uint32_t)kBuckets - 1);
                        // (the last bucket holds all that is below: in units of its own octave)
                        v = Weights::moved(v, min(n + (kBuckets / 8 - 1) * kSteps, 0));
                        __hip_atomic_fetch_add(&mass[bucket * kCopies + copy], fixed(v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                        if (counted) __hip_atomic_fetch_add(&count[bucket * kCopies + copy], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
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
                sum = wave_scan((double)m * fixed.unit * pow2(-(int)(threadIdx.x >> 3)));
                if (counted) c = wave_scan(c);
                if (lane == 63) {
                    sums[wave] = sum;
                    counts[wave] = c;
                }
                __syncthreads();
                for (int i = 0; i < wave; ++i) {
                    sum += sums[i];
                    c += counts[i];
                }
                tile.mass[threadIdx.x] = sum;
                if (counted) tile.count[threadIdx.x] = c;
            }
            if (threadIdx.x == kTileGroups - 1) {
                tile.heads[0].sum = sum;
                tile.heads[0].most = key;
            }
        }
    }
}

// ---- second launch --------------------------------------------------------------------------------

constexpr int kMostParts2048 = kMostParts * kTileWaves;
// CAP: places collected.
template <int CAP> struct SortedShared {
    static constexpr int kMost = CAP;
    uint64_t mass[kBuckets];  // of a digit
    uint32_t count[kBuckets];
    double row_mass[kBuckets];  // of a bucket of the row and all above it, in the top octave's units
    uint32_t row_count[kBuckets];
    uint64_t within[kMostParts];  // kept weights of a tile within the border's bucket
    uint16_t active[kMostParts];
    uint64_t few[64];
    uint32_t n, n_active, left;
    // what the first wavefront finds for all
    int bucket;
    uint64_t lo, hi;
    double before;  // weights, and number, of what is before the range
    uint32_t count_before;
    uint64_t border;
    double reach;  // weights up to the border
    // (last, as the largest: what lies behind 64 KB has no offset of its own in an instruction)
    union {
        uint64_t list[CAP];
        struct {  // (before there is a list: the row's buckets in up to four parts)
            double mass_part[4 * kBuckets];
            uint32_t count_part[4 * kBuckets];
        };
    };
};
struct Nothing {};
template <int MODE, int CAP> struct PickShared {
    double part[MODE == FEW ? 1 : MODE == SORTED ? kMostParts : kMostParts2048];  // kept weights of a tile (or of a wavefront's part of it), in units of the row's top octave
    int shift[MODE == SORTED || MODE == ANY ? kMostParts : 1];                    // by how many buckets a tile's top octave is below the row's
    double table[kSteps], place[16];
    int pick;
    double pick_before;
    union {
        std::conditional_t<MODE == FEW || MODE == ANY, TopShared<2048>, Nothing> top;
        std::conditional_t<MODE == SORTED || MODE == ANY, SortedShared<CAP>, Nothing> sorted;
    };
};

// Writes a row's answer.
__device__ __forceinline__ void answer(const SampleArgs& a, int64_t row, int64_t token, double logp) {
    if (a.token64) ((int64_t*)a.token)[row] = token;
    else ((int32_t*)a.token)[row] = (int32_t)token;
    a.logp[row] = (float)logp;
}

// A row that is cut by its size or by its weights, as the second launch sees it.
template <class T> struct Row {
    static constexpr int VEC = 16 / sizeof(T), N = 32 / VEC;  // vectors of a lane: a wavefront takes 2048 logits at a time
    LogitRow<T> x;
    const SampleTile* tiles;
    int n_tiles;
    Weights w;
    Fixed fixed;
    uint32_t most;
    float most_value;
    int index_bits;

    __device__ __forceinline__ uint64_t place(uint32_t key, uint32_t index) const { return ((uint64_t)key << index_bits) | ((1u << index_bits) - 1 - index); }
    __device__ __forceinline__ uint32_t key_at(uint64_t place) const { return (uint32_t)(place >> index_bits); }
    __device__ __forceinline__ uint32_t index_at(uint64_t place) const { return ((1u << index_bits) - 1) - ((uint32_t)place & ((1u << index_bits) - 1)); }
    __device__ __forceinline__ double weight(uint32_t key) const { return w.of(value_of<T>(key), most_value); }
    __device__ __forceinline__ int bucket(uint32_t key) const {
        return min(w.below_any(value_of<T>(key), most_value) / kBucketSteps, kBuckets - 1);
    }

    // The smallest key up to `most` of which `is` holds; it holds for `most`, and above any key of which it holds. For a wavefront, 64 keys at a time.
    template <class Is> __device__ __forceinline__ uint32_t first_key(Is&& is) const {
        uint32_t lo = kNegInfKey<T> - 1, hi = most;  // not of lo, of hi
#pragma clang loop unroll(disable)
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
    // The smallest key of a bucket and those above it.
    __device__ __forceinline__ uint32_t first_key_of(int b) const {
        if (b == kBuckets - 1) return kNegInfKey<T>;
        return first_key([&](uint32_t key) { return bucket(key) <= b; });
    }
    // The largest key of a bucket that the row has something in.
    __device__ __forceinline__ uint32_t last_key_of(int b) const { return bucket(most) == b ? most : first_key_of(b - 1) - 1; }

    // Calls f(first vector of a lane, its bits) for every 2048 logits of the tiles of s.active, a wavefront each: the bits tell which of a lane's 32 have keys in klo ... khi.
    template <class Q, class F> __device__ __forceinline__ void each_piece(const Q& s, uint32_t klo, uint32_t khi, F&& f) const {
        const int lane = threadIdx.x & 63, waves = blockDim.x >> 6, all = (int)s.n_active * kTileWaves, last = x.vecs() - 1;
        if (all == 0) return;
        auto first_vec = [&](int i) { return (s.active[min(i, all - 1) / kTileWaves] * kTileWaves + min(i, all - 1) % kTileWaves) * (64 * N) + lane; };
        // keys side by side are bits side by side, but for zeros, whose sign does not count
        const uint32_t zero = Bits<T>::sign;
        const bool plain = khi < zero || klo > zero;
        const uint32_t base = klo > zero ? klo & ~zero : ~khi & Bits<T>::all, width = khi - klo;
        const float vlo = value_of<T>(klo), vhi = value_of<T>(khi);
        Pack<T, VEC> next[N];
        int i = threadIdx.x >> 6, v = first_vec(i);
#pragma unroll
        for (int n = 0; n < N; ++n) next[n] = x.raw(min(v + n * 64, last));
#pragma clang loop unroll(disable)
        for (; i < all; i += waves) {
            uint32_t miss = 0;  // bit 31 - m for logit m of a lane (two-byte ones: bit 15 - m / 2 for even ones, 31 - m / 2 for odd ones)
            if (!plain) {
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const float e = Elem<T>::widen(next[n].v[j]);
                        const int m = n * VEC + j, bit = sizeof(T) == 2 ? (m & 1 ? 31 : 15) - m / 2 : 31 - m;
                        miss |= e >= vlo && e <= vhi ? 0 : 1u << bit;
                    }
            } else if constexpr (sizeof(T) == 2) {
                typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
                struct Words {
                    uint32_t w[4];
                };
                const u16x2 b2 = {(uint16_t)base, (uint16_t)base}, w2 = {(uint16_t)width, (uint16_t)width}, one = {1, 1};
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    const Words words = __builtin_bit_cast(Words, next[n]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const u16x2 d = __builtin_bit_cast(u16x2, words.w[j]) - b2, out = __builtin_elementwise_min(d, w2) ^ d;
                        miss = miss << 1 | __builtin_bit_cast(uint32_t, __builtin_elementwise_min(out, one));
                    }
                }
            } else {
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) miss = miss << 1 | (bits_of(next[n].v[j]) - base > width ? 1u : 0u);
            }
            const int here = v;
            v = first_vec(i + waves);
#pragma unroll
            for (int n = 0; n < N; ++n) next[n] = x.raw(min(v + n * 64, last));
            f(here, ~miss);
        }
    }
    // Where the logit of a bit lies.
    static __device__ __forceinline__ int element_of(int first_vec, int bit) {
        const int m = sizeof(T) == 2 ? 2 * (15 - (bit & 15)) + (bit >> 4) : 31 - bit;
        return (first_vec + m / VEC * 64) * VEC + m % VEC;
    }
    // Collects into s.list the places of a range of keys; s.n: how many, of which only as many as it holds are there.
    template <class Q> __device__ __forceinline__ void collect(Q& s, uint32_t klo, uint32_t khi) const {
        __syncthreads();
        if (threadIdx.x == 0) s.n = 0;
        __syncthreads();
        each_piece(s, klo, khi, [&](int first, uint32_t hits) {
            // (what lies outside the row)
            if ((first & ~63) * VEC < x.lead || (first - (int)(threadIdx.x & 63) + 64 * N) * VEC > x.end)
                for (uint32_t h = hits; h; h &= h - 1)
                    if (!x.holds(element_of(first, __builtin_ctz(h)))) hits &= ~(h & -h);
            const int mine = __builtin_popcount(hits), upto = wave_scan(mine);
            uint32_t from = 0;
            if ((threadIdx.x & 63) == 63 && upto) from = atomicAdd(&s.n, (uint32_t)upto);
            uint32_t at = lane_of(from, 63) + upto - mine;
            const uint32_t lane_at = (uint32_t)first << 5;  // (a vector's number is below 2^22)
            for (; hits; hits &= hits - 1, ++at)
                if (at < Q::kMost) s.list[at] = lane_at | __builtin_ctz(hits);
        });
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < min(s.n, (uint32_t)Q::kMost); i += blockDim.x) {
            const int e = element_of((int)((uint32_t)s.list[i] >> 5), (int)s.list[i] & 31);
            s.list[i] = place(key_of(x.base[e]), e - x.lead);
        }
        __syncthreads();
    }
    // Calls f(place, value) of every logit whose place is in lo ... hi.
    template <class Q, class F> __device__ __forceinline__ void sweep(const Q& s, uint64_t lo, uint64_t hi, F&& f) const {
        each_piece(s, key_at(lo), key_at(hi), [&](int first, uint32_t hits) {
            for (; hits; hits &= hits - 1) {
                const int e = element_of(first, __builtin_ctz(hits));
                if (!x.holds(e)) continue;
                const T value = x.base[e];
                const uint64_t at = place(key_of(value), e - x.lead);
                if (at >= lo && at <= hi) f(at, Elem<T>::widen(value));
            }
        });
    }
};

// The tiles that have logits in a bucket of the row.
template <class T, class Shared> __device__ __forceinline__ void find_active(const Row<T>& r, Shared& s, int bucket) {
    auto& q = s.sorted;
    __syncthreads();
    if (threadIdx.x == 0) q.n_active = 0;
    __syncthreads();
    for (int t = threadIdx.x; t < r.n_tiles; t += blockDim.x) {
        const int src = bucket - s.shift[t];
        // (of the last bucket anything may be there, also what weighs nothing)
        const bool on = bucket == kBuckets - 1 || (src >= 0 && r.tiles[t].mass[src] > (src ? r.tiles[t].mass[src - 1] : 0.0));
        if (on) q.active[atomicAdd(&q.n_active, 1u)] = (uint16_t)t;
    }
    __syncthreads();
}

// The border: the first place of the order at which the number of tokens reaches `k` (by_count) or their weights reach `target`. Returns the place, in s.sorted.reach the weights up to it. `listed`: the bucket whose logits s.sorted.list holds, all of them, q.n in number.
template <class T, class Shared> __device__ __forceinline__ uint64_t find_border(const Row<T>& r, Shared& s, bool by_count, uint32_t k, double target, int& listed) {
    auto& q = s.sorted;
    constexpr int kMostList = std::remove_reference_t<decltype(q)>::kMost;
    const int lane = threadIdx.x & 63;
    __syncthreads();
    if (threadIdx.x < 64) {
        // the first bucket at which it is reached; where rounding keeps the sum below the target, the last that adds anything
        int b = -1, last = 0;
        for (int c = 0; c < kBuckets / 64; ++c) {
            const int i = c * 64 + lane;
            const bool some = by_count ? q.row_count[i] > (i ? q.row_count[i - 1] : 0) : q.row_mass[i] > (i ? q.row_mass[i - 1] : 0.0);
            const uint64_t any = __ballot(some), reach = __ballot(some && (by_count ? q.row_count[i] >= k : q.row_mass[i] >= target));
            if (any) last = c * 64 + 63 - __builtin_clzll(any);
            if (b < 0 && reach) b = c * 64 + __builtin_ctzll(reach);
        }
        if (b < 0) b = last;
        const uint64_t lo = r.place(r.first_key_of(b), (1u << r.index_bits) - 1), hi = r.place(r.last_key_of(b), 0);
        if (lane == 0) {
            q.bucket = b;
            q.before = b ? q.row_mass[b - 1] : 0.0;
            q.count_before = b && by_count ? q.row_count[b - 1] : 0;
            q.lo = lo;
            q.hi = hi;
        }
    }
    __syncthreads();
    const int bucket = q.bucket;
    const double up = pow2(bucket >> 3), unit = pow2(-(bucket >> 3)) * r.fixed.unit;  // of the bucket's octave
    auto weight = [&](float x) { return r.fixed(r.w.of(x, r.most_value) * up); };
    // Sums that differ by a rounding may show something in an empty bucket (one without any key has its range upside down): what is before it reaches the target then.
    const bool none = q.lo > q.hi;
    if (!none && listed != bucket) {
        find_active(r, s, bucket);
        r.collect(q, r.key_at(q.lo), r.key_at(q.hi));
        listed = q.n <= kMostList ? bucket : -1;
    }
    if (none || q.n == 0) {
        if (threadIdx.x == 0) q.reach = q.before;
        __syncthreads();
        return q.hi + 1;
    }
    uint32_t n = q.n;
    bool have = n <= kMostList;
#pragma clang loop unroll(disable)
    while (true) {
        if (!have && n <= kMostList) {
            // (never reached with more than that: what is counted is what is found)
            __syncthreads();
            if (threadIdx.x == 0) q.n = 0;
            __syncthreads();
            r.sweep(q, q.lo, q.hi, [&](uint64_t at, float) { q.list[atomicAdd(&q.n, 1u) % kMostList] = at; });
            __syncthreads();
            have = true;
        }
        if (have && n <= 64) break;
        // by eight bits of the place
        for (int i = threadIdx.x; i < kBuckets; i += blockDim.x) {
            q.mass[i] = 0;
            q.count[i] = 0;
        }
        __syncthreads();
        const uint64_t lo = q.lo, hi = q.hi, width = hi - lo;
        const int bits = width ? 64 - __builtin_clzll(width) : 0, shift = bits > 8 ? bits - 8 : 0;
        auto count = [&](uint64_t at, float x) {
            const int d = 255 - (int)((at - lo) >> shift);  // (the largest first)
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
            r.sweep(q, lo, hi, count);
        }
        __syncthreads();
        if (threadIdx.x < 64) {
            // the first digit at which it is reached, or the last that there is, 64 digits at a time
            uint64_t mass = 0;
            uint32_t number = 0;
            int d = -1, last = 0;
            uint64_t mass_last = 0, mass_before = 0;
            uint32_t number_last = 0, number_before = 0;
            for (int c = 0; c < kBuckets / 64 && d < 0; ++c) {
                const uint64_t m = wave_scan(q.mass[c * 64 + lane]) + mass;
                const bool some = q.count[c * 64 + lane] > 0;
                const uint32_t n = wave_scan(q.count[c * 64 + lane]) + number;
                const uint64_t any = __ballot(some), reach = __ballot(some && (by_count ? q.count_before + n >= k : q.before + (double)m * unit >= target));
                const int at = reach ? __builtin_ctzll(reach) : any ? 63 - __builtin_clzll(any) : 0;
                // (what is before that digit)
                const uint64_t m0 = lane_of(m - q.mass[c * 64 + lane], at);
                const uint32_t n0 = lane_of(n - q.count[c * 64 + lane], at);
                if (any) {
                    last = c * 64 + at;
                    mass_last = m0;
                    number_last = n0;
                }
                if (reach) {
                    d = last;
                }
                mass = lane_of(m, 63);
                number = lane_of(n, 63);
            }
            mass_before = mass_last;
            number_before = number_last;
            wave_fence();
            if (lane == 0) {
                q.lo = lo + ((uint64_t)(255 - last) << shift);
                q.hi = min(hi, q.lo + ((1ull << shift) - 1));
                q.before += (double)mass_before * unit;
                q.count_before += number_before;
                q.left = q.count[last];
            }
        }
        __syncthreads();
        n = q.left;
    }
    // at most 64 are left: a lane each
    __syncthreads();
    if (threadIdx.x == 0) q.left = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < min(q.n, (uint32_t)kMostList); i += blockDim.x) {
        const uint64_t at = q.list[i];
        if (at >= q.lo && at <= q.hi) q.few[atomicAdd(&q.left, 1u) & 63] = at;
    }
    __syncthreads();
    if (threadIdx.x < 64) {
        const int left = min((int)q.left, 64);
        const uint64_t mine = lane < left ? q.few[lane] : 0;
        const uint64_t m = lane < left ? weight(value_of<T>(r.key_at(mine))) : 0;
        uint64_t upto = 0;
        uint32_t number = 0;
        for (int j = 0; j < left; ++j) {
            const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(mine >> 32), j) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)mine, j);
            const uint64_t om = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(m >> 32), j) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)m, j);
            if (other >= mine) {
                upto += om;
                ++number;
            }
        }
        const bool reached = lane < left && (by_count ? q.count_before + number >= k : q.before + (double)upto * unit >= target);
        // the first that reaches it, or the last there is
        const uint32_t score = reached ? 1024 - number : lane < left ? number : 0;
        const uint64_t best = __ballot(score == wave_max(score));
        wave_fence();
        if (lane == __builtin_ctzll(best)) {
            q.border = mine;
            q.reach = q.before + (double)upto * unit;
        }
    }
    __syncthreads();
    return q.border;
}

// u's token among the first k <= 2 * 64 of an order in LDS (key and index as place_of has them), for a wavefront; `weight`: as many numbers in LDS.
template <class T> __device__ __forceinline__ void pick_of_few(const SampleArgs& a, int64_t row, const Settings& set, const double* table, const uint64_t* order, double* weight, int k, double u) {
    const int lane = threadIdx.x & 63;
    const uint32_t most = key_of_place(order[0]);
    if (no_number<T>(most)) {
        if (lane == 0) answer(a, row, -1, __builtin_nan(""));
        return;
    }
    const Weights w(table, value_of<T>(most), set.steps);
    double v[2], sum = 0.0;
    uint32_t index[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint64_t at = lane * 2 + i < k ? order[lane * 2 + i] : 0;
        index[i] = index_of(at);
        v[i] = lane * 2 + i < k ? w.of(value_of<T>(key_of_place(at)), value_of<T>(most)) : 0.0;
        if (lane * 2 + i < k) weight[lane * 2 + i] = v[i];
        sum += v[i];
    }
    wave_fence();
    const double upto = wave_scan(sum), before = lane_before(upto);
    const double target = set.p * lane_of(upto, 63), least = fmin(set.least, 1.0) * lane_of(v[0], 0);
    // how many are kept
    int cut = k;
#pragma unroll
    for (int i = 1; i >= 0; --i) {
        const int at = lane * 2 + i;
        const double here = i ? before + sum : before + v[0];
        if (at >= k) continue;
        if (set.p < 1.0 && here >= target) cut = at + 1;
        if (v[i] < least && at > 0) cut = at;
    }
    struct MinI {
        __device__ static __forceinline__ int comb(int a, int b) { return min(a, b); }
    };
    const int kept = group_reduce<MinI>(cut, 64);
    const double whole = lane_of(((kept - 1) & 1) ? before + sum : before + v[0], (kept - 1) >> 1);
    // u's token: the last by index whose weights before it do not exceed u's part
    const double part = u * whole;
    double s0 = 0.0, s1 = 0.0;
#pragma unroll 4
    for (int j = 0; j < kept; ++j) {
        const uint32_t other = index_of(order[j]);
        const double o = weight[j];
        s0 += other < index[0] ? o : 0.0;
        s1 += other < index[1] ? o : 0.0;
    }
    uint32_t token = 0;
    if (lane * 2 < kept && v[0] > 0.0 && s0 <= part) token = index[0] + 1;
    if (lane * 2 + 1 < kept && v[1] > 0.0 && s1 <= part) token = max(token, index[1] + 1);
    const uint32_t best = wave_max(token);
    if (token == best && best) answer(a, row, best - 1, log((index[0] + 1 == best ? v[0] : v[1]) / whole));
}

// THREADS: at most. Few rows have larger workgroups, and room for more of a bucket.
template <class T, int MODE, int THREADS>
__global__ __launch_bounds__(THREADS, THREADS == 1024 ? 4 : MODE == SORTED ? 3 : 1) void sample_pick_kernel(const SampleArgs a, const Settings all_rows, int64_t row0, int64_t rows) {
    constexpr int VEC = 16 / sizeof(T);
    __shared__ PickShared<MODE, THREADS == 1024 ? 8192 : 4096> s;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    make_table(s.table);
    for (int64_t at = blockIdx.x; at < rows; at += gridDim.x) {
        const int64_t row = row0 + at;
        __syncthreads();
        const LogitRow<T> x((const T*)a.x + offset_of(a.kept, row), a.cols);
        const SampleTile* tiles = (const SampleTile*)a.tiles_scratch + at * a.tiles;
        const Settings set = Settings::of<MODE>(a, all_rows, row);
        const int mode = MODE == ANY ? set.mode : MODE;
        double u = a.u[row];
        u = u > 0.0 ? u : 0.0;
        if (mode == BAD) {
            if (threadIdx.x == 0) answer(a, row, -1, __builtin_nan(""));
            continue;
        }
        if constexpr (MODE == FEW || MODE == ANY) {
            if (mode == FEW) {
                const int k = set.k;
                const int n = collect_top(s.top, x, tiles->keys, a.tiles, k, sizeof(SampleTile));
                uint64_t* order = (uint64_t*)s.top.groups;
                static_assert(sizeof s.top.groups >= kMostTop * sizeof(uint64_t), "");
                rank_top(s.top, n, k, [&](int rank, uint64_t p) { order[rank] = p; });
                __syncthreads();
                double* weight = (double*)s.top.list;
                static_assert(sizeof s.top.list >= kMostTop * sizeof(double), "");
                if (k <= 128) {
                    if (wave == 0) pick_of_few<T>(a, row, set, s.table, order, weight, k, u);
                    continue;
                }
                const uint32_t most = key_of_place(order[0]);
                if (no_number<T>(most)) {
                    if (threadIdx.x == 0) answer(a, row, -1, __builtin_nan(""));
                    continue;
                }
                const Weights w(s.table, value_of<T>(most), set.steps);
                const int each = (k + (int)blockDim.x - 1) / (int)blockDim.x, i0 = min((int)threadIdx.x * each, k), i1 = min(i0 + each, k);
                double mine = 0.0;
                for (int i = i0; i < i1; ++i) mine += weight[i] = w.of(value_of<T>(key_of_place(order[i])), value_of<T>(most));
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
                __syncthreads();
                // u's token, by eight bits of the index at a time, from sums of whole numbers of 2^-50, which have no order (every wavefront looks for itself)
                const double part = u * s.pick_before;
                uint64_t* mass = (uint64_t*)s.top.digits.n;
                static_assert(sizeof s.top.digits.n >= 256 * sizeof(uint64_t), "");
                uint32_t prefix = 0;
                uint64_t upto_prefix = 0;
#pragma clang loop unroll(disable)
                for (int shift = a.cols > 1 << 16 ? 16 : a.cols > 1 << 8 ? 8 : 0; shift >= 0; shift -= 8) {
                    for (int i = threadIdx.x; i < 256; i += blockDim.x) mass[i] = 0;
                    __syncthreads();
                    for (int i = threadIdx.x; i < kept; i += blockDim.x) {
                        const uint32_t index = index_of(order[i]);
                        if (index >> (shift + 8) == prefix)
                            __hip_atomic_fetch_add(&mass[index >> shift & 255], __builtin_bit_cast(uint64_t, weight[i] + 4.0) - __builtin_bit_cast(uint64_t, 4.0), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                    }
                    __syncthreads();
                    // the first digit at which the sum exceeds u's part, or the last that has something
                    uint64_t m[4], sum = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        m[i] = mass[lane * 4 + i];
                        sum += m[i];
                    }
                    const uint64_t end = wave_scan(sum) + upto_prefix;
                    const uint64_t over = __ballot(sum > 0 && (double)end * 0x1p-50 > part), some = __ballot(sum > 0);
                    const int l = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(some);
                    uint64_t before = end - sum, from = before;
                    int digit = 0;
                    bool done = false;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (m[i] > 0 && !done) {
                            digit = lane * 4 + i;
                            from = before;
                            done = (double)(before + m[i]) * 0x1p-50 > part;
                        }
                        before += m[i];
                    }
                    prefix = prefix << 8 | lane_of((uint32_t)digit, l);
                    upto_prefix = lane_of(from, l);
                    __syncthreads();
                }
                for (int i = threadIdx.x; i < kept; i += blockDim.x)
                    if (index_of(order[i]) == prefix) answer(a, row, prefix, log(weight[i] / s.pick_before));
                continue;
            }
        }
        if constexpr (MODE != FEW) {
            // the parts together (every wavefront for itself): tiles, or a wavefront's 2048 logits of one
            const int per = MODE == PLAIN || mode == PLAIN ? kTileWaves : 1, parts = a.tiles * per;
            auto head = [&](int t) -> const SampleHead& { return tiles[t / per].heads[t % per]; };
            uint32_t most = 0;
            for (int t = lane; t < parts; t += 64) most = max(most, head(t).most);
            most = wave_max(most);
            if (no_number<T>(most)) {
                if (threadIdx.x == 0) answer(a, row, -1, __builtin_nan(""));
                continue;
            }
            const float most_value = value_of<T>(most);
            Row<T> r{x, tiles, a.tiles, Weights(s.table, most_value, set.steps), Fixed(a.cols), most, most_value, a.cols > 1 ? 32 - __builtin_clz((unsigned)a.cols - 1) : 0};
            uint64_t border = 0;
            for (int t = threadIdx.x; t < parts; t += blockDim.x) {
                const uint32_t key = head(t).most;
                int shift = 1 << 20;
                double part = 0.0;
                if (key > kNegInfKey<T>) {
                    const float v = value_of<T>(key);
                    // (what a part's largest is 96 octaves below weighs nothing, here as for a single logit)
                    if (((double)most_value - (double)v) * r.w.steps < 96.0 * kSteps) {
                        shift = -(r.w.above(v) >> 7) * 8;
                        part = head(t).sum * pow2(-(shift >> 3));
                    }
                }
                if (MODE != PLAIN && per == 1) s.shift[t] = shift;
                s.part[t] = part;
            }
            if constexpr (MODE == SORTED || MODE == ANY) {
                if (mode == SORTED) {
                    auto& q = s.sorted;
                    const bool counted = set.k < a.cols;
                    __syncthreads();
                    // the row's buckets: those of its tiles, dealt to up to four threads a bucket
                    const int quarters = blockDim.x / kBuckets, b = threadIdx.x % kBuckets;
                    double mine = 0.0;
                    uint32_t number = 0;
#pragma unroll 8
                    for (int t = threadIdx.x / kBuckets; t < a.tiles; t += quarters) {
                        const int shift = s.shift[t], src = max(b - shift, 0);
                        const double m = tiles[t].mass[src];
                        mine += b >= shift ? m * pow2(-min(shift >> 3, 1000)) : 0.0;
                    }
                    if (counted)
#pragma unroll 8
                        for (int t = threadIdx.x / kBuckets; t < a.tiles; t += quarters) {
                            const int shift = s.shift[t];
                            const uint32_t c = tiles[t].count[max(b - shift, 0)];
                            number += b >= shift ? c : 0;
                        }
                    q.mass_part[threadIdx.x] = mine;
                    q.count_part[threadIdx.x] = number;
                    double all = 0.0;  // (the same in every wavefront)
                    for (int t = lane; t < a.tiles; t += 64) all += s.part[t];
                    all = group_reduce<SumD>(all, 64);
                    __syncthreads();
                    if (threadIdx.x < kBuckets) {
                        for (int i = 1; i < quarters; ++i) {
                            mine += q.mass_part[threadIdx.x + i * kBuckets];
                            number += q.count_part[threadIdx.x + i * kBuckets];
                        }
                        // (the last bucket has all the rest)
                        q.row_mass[threadIdx.x] = b == kBuckets - 1 ? all : fmin(mine, all);
                        q.row_count[threadIdx.x] = b == kBuckets - 1 ? (uint32_t)a.cols : number;
                    }
                    int listed = -1;
                    double whole = all;
#pragma clang loop unroll(disable)
                    for (int by = counted ? 0 : 1; by < (set.p < 1.0 ? 2 : 1); ++by) {
                        border = max(border, find_border(r, s, by == 0, set.k, set.p * whole, listed));
                        if (by == 0) whole = q.reach;
                    }
                    __syncthreads();
                    if (wave == 0) {
                        if (set.least > 0.0) {
                            const double least = fmin(set.least, 1.0) * r.weight(most);
                            border = max(border, (uint64_t)r.first_key([&](uint32_t key) { return r.weight(key) >= least; }) << r.index_bits);
                        }
                        const int bucket = border ? r.bucket(r.key_at(border)) : 0;
                        const uint32_t khi = r.last_key_of(bucket);
                        if (lane == 0) {
                            q.border = border;
                            q.bucket = bucket;
                            q.hi = r.place(khi, 0);
                        }
                    }
                    for (int t = threadIdx.x; t < a.tiles; t += blockDim.x) q.within[t] = 0;
                    __syncthreads();
                    border = q.border;
                    if (border) {
                        // what is kept of each tile: its buckets above the border's, and within that bucket the logits up to the border
                        const int bucket = q.bucket;
                        const double up = pow2(bucket >> 3);
                        auto add = [&](uint64_t at, float v) {
                            __hip_atomic_fetch_add(&q.within[(r.index_at(at) + x.lead) / kTile], r.fixed(r.w.of(v, most_value) * up), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                        };
                        if (listed == bucket) {
                            for (uint32_t i = threadIdx.x; i < q.n; i += blockDim.x) {
                                const uint64_t p = q.list[i];
                                if (p >= border) add(p, value_of<T>(r.key_at(p)));
                            }
                        } else {
                            find_active(r, s, bucket);
                            r.sweep(q, border, q.hi, add);
                        }
                        __syncthreads();
                        for (int t = threadIdx.x; t < a.tiles; t += blockDim.x) {
                            const int shift = s.shift[t], src = bucket - 1 - shift;
                            const double above = src >= 0 ? tiles[t].mass[src] * pow2(-(shift >> 3)) : 0.0;
                            s.part[t] = above + (double)q.within[t] * (pow2(-(bucket >> 3)) * r.fixed.unit);
                        }
                    }
                }
            }
            __syncthreads();
            // u's part: the first at which the sum exceeds u of the whole (every wavefront for itself; a lane has the parts from t0 on)
            const int each = (parts + 63) / 64, t0 = min(lane * each, parts), t1 = min(t0 + each, parts);
            double mine = 0.0;
            for (int t = t0; t < t1; ++t) mine += s.part[t];
            const double upto = wave_scan(mine), whole = lane_of(upto, 63), target = u * whole;
            const uint64_t above = __ballot(mine > 0.0 && upto > target), some = __ballot(mine > 0.0);
            const int owner = above ? __builtin_ctzll(above) : 63 - __builtin_clzll(some);
            double before = lane_before(upto);
            int part = t0;
            for (int t = t0, last = -1; t < t1; ++t) {
                if (s.part[t] > 0.0) {
                    if (last >= 0) before += s.part[last];
                    part = t;
                    if (before + s.part[t] > target) break;
                    last = t;
                }
            }
            part = lane_of(part, owner);
            const double rest = fmax(target - lane_of(before, owner), 0.0);
            // and its token there: a thread has `run` neighbours of the part
            const int size = kTile / per, run = max(size / (int)blockDim.x, VEC), e0 = part * size + (int)threadIdx.x * run;
            mine = 0.0;
#pragma clang loop unroll(disable)
            for (int v = e0 / VEC; v < (e0 + run) / VEC; ++v) {
                if (v > x.vecs() - 1 || e0 >= (part + 1) * size) break;
                const Pack<T, VEC> p = x.raw(v);
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const int e = v * VEC + i;
                    const bool on = x.holds(e) && r.place(key_of(p.v[i]), e - x.lead) >= border;
                    mine += on ? r.w.of(Elem<T>::widen(p.v[i]), most_value) : 0.0;
                }
            }
            double whole_part;
            const double here = scan_before(mine, s.place, whole_part);
            // The wavefront in which the sum crosses it and the first thread there that does, or the last that has something (the sum over the part may be a rounding off what it was chosen by).
            // Every wavefront looks at the same numbers, so one answers. (Sums up to a wavefront are a tree's, which behind the last weight may still rise by a rounding.)
            const double wave_sum = lane < waves ? s.place[lane] : 0.0, wave_upto = wave_scan(wave_sum);
            const uint64_t beyond = __ballot(wave_sum > 0.0 && wave_upto > rest), weighty = __ballot(wave_sum > 0.0);
            if (wave == (beyond ? __builtin_ctzll(beyond) : weighty ? 63 - __builtin_clzll(weighty) : 0)) {
                const uint64_t crosses = __ballot(mine > 0.0 && here + mine > rest), some = __ballot(mine > 0.0);
                const int l = crosses ? __builtin_ctzll(crosses) : some ? 63 - __builtin_clzll(some) : 0;
                const int e = lane_of(e0, l) + lane;
                double w = 0.0;
                if (lane < run && x.holds(e)) {
                    const T v = x.base[e];
                    if (r.place(key_of(v), e - x.lead) >= border) w = r.w.of(Elem<T>::widen(v), most_value);
                }
                const double from = lane_of(here, l), sum = wave_scan(w);
                const uint64_t over = __ballot(w > 0.0 && from + sum > rest), any = __ballot(w > 0.0);
                const int pick = over ? __builtin_ctzll(over) : any ? 63 - __builtin_clzll(any) : 0;
                if (lane == pick) answer(a, row, e - x.lead, log(fmin(w / whole, 1.0)));
            }
        }
    }
}

// A wavefront for each row, of which at most kWaveTop places matter. One of which it would collect too much is left to the workgroup.
template <class T>
__global__ __launch_bounds__(kTileGroups) void sample_wave_kernel(const SampleArgs a, const Settings set, int64_t row0, int64_t rows) {
    constexpr int N = kTileGroups / 64;
    __shared__ union {
        WaveShared wave[N];
        TopShared<512> all;
    } s;
    __shared__ uint64_t order[N][kWaveTop];
    __shared__ double weight[N][kWaveTop], table[kSteps];
    __shared__ int left[N];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    make_table(table);
    __syncthreads();
    for (int64_t r0 = (int64_t)blockIdx.x * N; r0 < rows; r0 += (int64_t)gridDim.x * N) {
        const int64_t r = r0 + wave;
        auto keys_of = [&](int64_t r) { return ((const SampleTile*)a.tiles_scratch + r * a.tiles)->keys; };
        auto row_of = [&](int64_t r) { return LogitRow<T>((const T*)a.x + offset_of(a.kept, row0 + r), a.cols); };
        int n = 0;
        if (r < rows) {
            n = wave_top(s.wave[wave], row_of(r), keys_of(r), a.tiles, set.k, sizeof(SampleTile));
            if (n >= 0) wave_rank(s.wave[wave], n, set.k, [&](int rank, uint64_t p) { order[wave][rank] = p; });
        }
        if (lane == 0) left[wave] = n < 0;
        __syncthreads();
        for (int w = 0; w < N; ++w) {
            if (!left[w]) continue;
            const int all = collect_top(s.all, row_of(r0 + w), keys_of(r0 + w), a.tiles, set.k, sizeof(SampleTile));
            rank_top(s.all, all, set.k, [&](int rank, uint64_t p) { order[w][rank] = p; });
            __syncthreads();
        }
        if (r < rows) {
            const double u = a.u[row0 + r];
            pick_of_few<T>(a, row0 + r, set, table, order[wave], weight[wave], set.k, u > 0.0 ? u : 0.0);
        }
        __syncthreads();
    }
}

}  // namespace

size_t sample_row_bytes(int dtype, int64_t cols) { return (size_t)tiles_of(dtype, cols, true) * sizeof(SampleTile); }

void launch_sample(int dtype, const SampleArgs& a, hipStream_t st) {
    static_assert(sizeof(SampleTile) % 16 == 0, "every tile's keys are aligned");
    const bool each = a.temperature.each || a.top_k.each || a.top_p.each || a.min_p.each;
    const Settings set(a.temperature.all, a.top_k.all, a.top_p.all, a.min_p.all, a.cols);
    HPT_WITH_TYPE(dtype, {
        for (int64_t row0 = 0; row0 < a.rows; row0 += a.run) {
            const int64_t rows = std::min(a.run, a.rows - row0);
            const unsigned blocks = (unsigned)rows;
            // (beyond a workgroup for each compute unit, smaller ones, several to a unit. bf16 [200, 50257] and [500, 50257], top_p 0.9, us: 48.8 and 91.9 with 1024 threads, 49.8 and 72.8 with 256)
            const bool many = rows > 256;
            auto both = [&](auto mode) {
                constexpr int MODE = decltype(mode)::value;
                sample_tiles_kernel<T, MODE><<<dim3((unsigned)a.tiles, blocks), kTileGroups, 0, st>>>(a, set, row0);
                if constexpr (MODE == PLAIN) {
                    sample_pick_kernel<T, MODE, 256><<<blocks, 256, 0, st>>>(a, set, row0, rows);
                } else {
                    if constexpr (MODE == FEW)
                        if (for_a_wave<T>(rows, a.tiles, set.k)) return sample_wave_kernel<T><<<(blocks + 3) / 4, kTileGroups, 0, st>>>(a, set, row0, rows);
                    if constexpr (MODE != FEW)
                        if (many) return sample_pick_kernel<T, MODE, 256><<<blocks, 256, 0, st>>>(a, set, row0, rows);
                    sample_pick_kernel<T, MODE, 1024><<<blocks, many ? 256 : 1024, 0, st>>>(a, set, row0, rows);
                }
            };
            if (each) both(std::integral_constant<int, ANY>{});
            else if (set.mode == FEW) both(std::integral_constant<int, FEW>{});
            else if (set.mode == PLAIN) both(std::integral_constant<int, PLAIN>{});
            else both(std::integral_constant<int, SORTED>{});
        }
    });
}

}  // namespace hpt
