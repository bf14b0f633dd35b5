// The k largest logits of each row, in order, and the log of the sum of exponentials of the row over a temperature.
//
// Two launches. The first reads the logits once, in tiles of 8192: the largest key of each 32 neighbours stays (and, where the sum is wanted, a wavefront
// adds the exponentials of its 2048 below their largest). The second has a workgroup for each row, which finds the first k places from those keys (top_rows.hpp).
// The second is bound by the latency of its steps.
//
// The first reads bf16 [4096, 50257] in 71 to 73 us (5.7 TB/s) without the sum; with it the launch is bound by its instructions, six for each logit: 94 to 102 us (4.2 TB/s; f32 148 to 153, 5.5 TB/s). The second takes 32 to 36
// of k = 64 there (by wavefronts), 9 of one row of 152000 and of 37 of 50257, 19 of f16 [256, 152000] with k = 512, where the first places lie in an octave or two (top_rows.hpp has the others). Small rows have a launch of their own.
#include <algorithm>
#include <cmath>

#include "top_rows.hpp"

namespace hpt {

Steps steps_of(double temperature) {
    const double a = 1.4426950408889634 / temperature;
    int e;
    const double m = std::frexp(a, &e);
    Steps s;
    s.hi = (float)std::ldexp((std::ceil(m * 4096.0) - 1.0) / 4096.0, e);
    s.lo = (float)(a - (double)s.hi);
    return s;
}

int64_t tiles_of(int dtype, int64_t cols, bool shifted) { return (cols + (shifted ? 16 / (int64_t)dtype_size(dtype) - 1 : 0) + kTile - 1) / kTile; }
bool rows_shifted(int dtype, const void* x, const Dims& kept) {
    bool aligned = (uintptr_t)x % 16 == 0;
    for (int i = 0; i < kept.n; ++i) aligned = aligned && kept.stride[i] * (int64_t)dtype_size(dtype) % 16 == 0;
    return !aligned;
}
// (as many as a launch's second dim takes, too)
int64_t rows_of_run(int64_t rows, size_t row_bytes) { return std::max<int64_t>(1, std::min<int64_t>({rows, 32768, (int64_t)(kMostRowScratch / row_bytes)})); }
size_t topk_row_bytes(int dtype, int64_t cols, bool lse) {
    return (size_t)tiles_of(dtype, cols, true) * (kTileGroups * dtype_size(dtype) + (lse ? kTileWaves * 2 * sizeof(double) : 0));
}

namespace {

constexpr int kMostList = 2048;

template <class T, bool LSE>
__global__ __launch_bounds__(kTileGroups) void topk_groups_kernel(const TopkArgs a, int64_t row0) {
    constexpr int VEC = 16 / sizeof(T), V = kTileVecs<T>;
    const int64_t row = blockIdx.y;
    for (int tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
        const int64_t at = row * a.tiles + tile;
        Pack<T, VEC> p[V];
        load_tile<T>(LogitRow<T>((const T*)a.x + offset_of(a.kept, row0 + row), a.cols), tile, p);
        const uint32_t key = group_key<T>(p);
        ((KeyOf<T>*)a.keys)[at * kTileGroups + threadIdx.x] = (KeyOf<T>)key;
        if constexpr (LSE) {
            // a wavefront's part of the sum, below its own largest: in 32 bits within a vector, by twos, in 64 beyond. (Exponents from log2 e / temperature in two pieces: as one f32
            // it would be 2^-25 of a distance D off itself, and all terms at D with it.)
            const uint32_t top = wave_max(key);
            double part = 0.0;
            // (NaN, +inf and nothing but -inf are told from the largest alone)
            const bool number = top < kInfKey<T> && top > kNegInfKey<T>;
            const float most = number ? value_of<T>(top) : top == kInfKey<T> ? __builtin_huge_valf() : top <= kNegInfKey<T> ? -__builtin_huge_valf() : __builtin_nanf("");
            if (number) {
#pragma unroll
                for (int b = 0; b < V; ++b) {
                    float e[VEC];
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        const float d = Elem<T>::widen(p[b].v[i]) - most;
                        e[i] = __builtin_amdgcn_exp2f(fmaf(d, a.steps.hi, d * a.steps.lo));
                    }
                    part += (double)sum_by_twos(e);
                }
            }
            const double sum = group_reduce<SumD>(part, 64);
            if ((threadIdx.x & 63) == 0) {
                double* to = a.sums + (at * kTileWaves + (threadIdx.x >> 6)) * 2;
                to[0] = most;
                to[1] = sum;
            }
        }
    }
}

// What a row's k places become.
template <class T> struct Answer {
    const TopkArgs& a;
    const T* x;
    int64_t row;
    __device__ __forceinline__ void operator()(int rank, uint64_t at) const {
        const uint32_t i = index_of(at), key = key_of_place(at);
        // (a key tells the logit, but for zeros' signs and NaNs' bits)
        ((T*)a.values)[row * a.k + rank] = key == Bits<T>::sign || key == kNanKey<T> ? x[i] : Elem<T>::narrow(value_of<T>(key));
        if (a.index64) ((int64_t*)a.index)[row * a.k + rank] = i;
        else ((int32_t*)a.index)[row * a.k + rank] = (int32_t)i;
    }
};
// The largest logit of a row and its sum of exponentials below that, from the row's parts, for a wavefront. Parts are weighted by the hardware's exponential of a fraction (two half steps), and by whole octaves.
struct RowSum {
    double most, sum;
};
__device__ __forceinline__ RowSum sum_of_parts(const TopkArgs& a, const double* p) {
    const int lane = threadIdx.x & 63, parts = a.tiles * kTileWaves;
    const double inf = __builtin_huge_val(), steps = 1.4426950408889634 * a.inv_temperature;
    // (a lane's first part stays; those of longer rows are fetched again)
    const bool any = lane < parts;
    const double most0 = any ? p[2 * lane] : -inf, part0 = any ? p[2 * lane + 1] : 0.0;
    double all = most0;
    bool nan = most0 != most0;
    for (int t = lane + 64; t < parts; t += 64) {
        const double most = p[2 * t];
        nan |= most != most;
        all = fmax(all, most);
    }
#pragma unroll
    for (int w = 1; w < 64; w <<= 1) all = fmax(all, shfl_xor_any(all, w));
    auto share = [&](double most, double part) {
        const double d = fmax((most - all) * steps, -1000.0), whole = rint(d);
        return part > 0.0 ? part * ldexp((double)__builtin_amdgcn_exp2f((float)(d - whole)), (int)whole) : 0.0;
    };
    double sum = share(most0, part0);
    for (int t = lane + 64; t < parts; t += 64) sum += share(p[2 * t], p[2 * t + 1]);
    sum = group_reduce<SumD>(sum, 64);
    return {__any(nan) ? __builtin_nan("") : all, sum};
}
// The logarithm is one of 64 bits: what is off in lse are the parts' roundings, some 2^-24 of the sum whatever lse's own size, and its own one. (32 bits of it would be 2^-24 of the logarithm, of which
// little may be left in lse: of log-probabilities, nothing.)
__device__ __forceinline__ void store_lse(const TopkArgs& a, const RowSum& s, int64_t row) {
    a.lse[row] = (float)(s.most * a.inv_temperature + (fabs(s.most) < __builtin_huge_val() ? log(s.sum) : 0.0));
}

// A workgroup for each row.
template <class T, bool LSE>
__global__ __launch_bounds__(1024) void topk_pick_kernel(const TopkArgs a, int64_t row0, int64_t rows) {
    __shared__ TopShared<kMostList> s;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T* x = (const T*)a.x + offset_of(a.kept, row0 + r);
        const int n = collect_top(s, LogitRow<T>(x, a.cols), (const KeyOf<T>*)a.keys + r * a.tiles * kTileGroups, a.tiles, a.k, kTileGroups * sizeof(T));
        rank_top(s, n, a.k, Answer<T>{a, x, row0 + r});
        // (the last wavefront has fewest places to rank)
        if (LSE && threadIdx.x >= blockDim.x - 64) {
            const RowSum sum = sum_of_parts(a, a.sums + 2 * r * a.tiles * kTileWaves);
            if (threadIdx.x == blockDim.x - 64) store_lse(a, sum, row0 + r);
        }
        __syncthreads();
    }
}

// A wavefront for each row, few places. A row of which it would collect too much is left to the workgroup. (As many wavefronts of a SIMD as LDS has room for.)
template <class T, bool LSE>
__global__ __launch_bounds__(kTileGroups, 5) void topk_wave_kernel(const TopkArgs a, int64_t row0, int64_t rows) {
    constexpr int N = kTileGroups / 64;
    __shared__ union {
        WaveShared wave[N];
        TopShared<512> all;
    } s;
    static_assert(kWaveTop <= 512, "the first k fit the list");
    __shared__ int left[N];
    __shared__ RowSum sums[LSE ? N : 1];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int64_t r0 = (int64_t)blockIdx.x * N; r0 < rows; r0 += (int64_t)gridDim.x * N) {
        const int64_t r = r0 + wave;
        int n = 0;
        if (r < rows) {
            const T* x = (const T*)a.x + offset_of(a.kept, row0 + r);
            n = wave_top(s.wave[wave], LogitRow<T>(x, a.cols), (const KeyOf<T>*)a.keys + r * a.tiles * kTileGroups, a.tiles, a.k, kTileGroups * sizeof(T));
            if (n >= 0) wave_rank(s.wave[wave], n, a.k, Answer<T>{a, x, row0 + r});
            if constexpr (LSE) {
                const RowSum sum = sum_of_parts(a, a.sums + 2 * r * a.tiles * kTileWaves);
                if ((threadIdx.x & 63) == 0) sums[wave] = sum;
            }
        }
        if ((threadIdx.x & 63) == 0) left[wave] = n < 0;
        __syncthreads();
        // (logarithms of the workgroup's rows side by side, a lane each)
        if (LSE && threadIdx.x < N && r0 + threadIdx.x < rows) store_lse(a, sums[LSE ? threadIdx.x : 0], row0 + r0 + threadIdx.x);
        for (int w = 0; w < N; ++w) {
            if (!left[w]) continue;
            const T* x = (const T*)a.x + offset_of(a.kept, row0 + r0 + w);
            const int all = collect_top(s.all, LogitRow<T>(x, a.cols), (const KeyOf<T>*)a.keys + (r0 + w) * a.tiles * kTileGroups, a.tiles, a.k, kTileGroups * sizeof(T));
            rank_top(s.all, all, a.k, Answer<T>{a, x, row0 + r0 + w});
            __syncthreads();
        }
        __syncthreads();
    }
}

constexpr int kMostEach = 4;  // rows of a wavefront
// Rows of at most 64 N elements, a wavefront each, one launch: the row stays in registers (element i of lane l is at 64 i + l), and the largest is taken out k times.
template <class T, int N, bool LSE>
__global__ __launch_bounds__(256) void topk_small_kernel(const TopkArgs a, int rows_each) {
    const int each = LSE ? rows_each : 1;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    __shared__ RowSum sums[LSE ? 4 * kMostEach : 1];
    for (int64_t row0 = (int64_t)blockIdx.x * 4 * each; row0 < a.rows; row0 += (int64_t)gridDim.x * 4 * each) {
        for (int n = 0; n < each; ++n) {
            const int64_t row = row0 + n * 4 + wave;
            if (row >= a.rows) break;
            const T* x = (const T*)a.x + offset_of(a.kept, row);
            T v[N];
            uint32_t key[N];
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = x[min(i * 64 + lane, a.cols - 1)];
#pragma unroll
            for (int i = 0; i < N; ++i) key[i] = i * 64 + lane < a.cols ? key_of(v[i]) : 0;
            uint32_t best = 0;
            int which = 0;
            auto find = [&] {
                best = 0;
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (key[i] > best) {
                        best = key[i];
                        which = i;
                    }
            };
            find();
            if constexpr (LSE) {
                // (as the groups' launch has it)
                constexpr int M = N < 4 ? N : 4;
                const uint32_t top = wave_max(best);
                const bool number = top < kInfKey<T> && top > kNegInfKey<T>;
                const float most = number ? value_of<T>(top) : top == kInfKey<T> ? __builtin_huge_valf() : top <= kNegInfKey<T> ? -__builtin_huge_valf() : __builtin_nanf("");
                double part = 0.0;
#pragma unroll
                for (int i = 0; i < N; i += M) {
                    float e[M];
#pragma unroll
                    for (int j = 0; j < M; ++j) {
                        const float d = Elem<T>::widen(v[i + j]) - most;
                        e[j] = (i + j) * 64 + lane < a.cols ? __builtin_amdgcn_exp2f(fmaf(d, a.steps.hi, d * a.steps.lo)) : 0.0f;
                    }
                    part += (double)sum_by_twos(e);
                }
                const double sum = group_reduce<SumD>(part, 64);
                if (lane == 0) sums[n * 4 + wave] = {most, sum};
            }
            uint32_t mine = 0, at = 0;
#pragma clang loop unroll(disable)
            for (int r = 0; r < a.k; ++r) {
                const uint32_t first = wave_max(best);
                const uint64_t who = __ballot(best == first);
                int l = __builtin_ctzll(who);
                if (who & (who - 1)) l = (int)(~wave_max(best == first ? ~(uint32_t)(which * 64 + lane) : 0u) & 63);  // (equal ones: the first)
                const uint32_t index = (uint32_t)lane_of(which, l) * 64 + l;
                if (lane == r) {
                    mine = first;
                    at = index;
                }
                const int gone = lane == l ? which : -1;
#pragma unroll
                for (int i = 0; i < N; ++i) key[i] = i == gone ? 0 : key[i];
                find();
            }
            if (lane < a.k) Answer<T>{a, x, row}(lane, place_of(mine, at));
        }
        if constexpr (LSE) {
            // (logarithms of the workgroup's rows side by side)
            __syncthreads();
            if (threadIdx.x < 4 * each && row0 + threadIdx.x < a.rows) store_lse(a, sums[threadIdx.x], row0 + threadIdx.x);
            __syncthreads();
        }
    }
}

}  // namespace

// Which rows topk_small_kernel takes (us, f32, against the two launches). Few rows, where a wavefront's steps stand one behind the other: [1, 2000] of k 8 10.0 / 10.4, of 20 18.6 / 11.1, [1, 256] of 64 12.9 / 14.2.
// Many: [500, 2000] of 20 19.9 / 20.2, of 64 52 / 70; a router's [16384, 64] of 8 7.8 / 132, [16384, 1000] of 64 161 / 717.
bool topk_in_registers(int64_t rows, int64_t cols, int64_t k) { return cols <= 64 * 32 && k <= 64 && (rows > 256 || k * ((cols + 63) / 64) <= 256); }

void launch_topk(int dtype, const TopkArgs& a, hipStream_t st) {
    HPT_WITH_TYPE(dtype, {
        if (topk_in_registers(a.rows, a.cols, a.k)) {
            auto small = [&](auto n, auto lse) {
                // (rows' logarithms side by side, with lse: f32 [100000, 64], k = 8, 42.5 us of four rows a wavefront and 46.5 of one, [16384, 64] 10.5 and 10.2)
                const int each = decltype(lse)::value && a.rows > 32768 ? kMostEach : 1;
                topk_small_kernel<T, decltype(n)::value, decltype(lse)::value><<<(unsigned)std::min<int64_t>((a.rows + 4 * each - 1) / (4 * each), 1 << 20), 256, 0, st>>>(a, each);
            };
            auto sized = [&](auto lse) {
                if (a.cols <= 64) small(std::integral_constant<int, 1>{}, lse);
                else if (a.cols <= 256) small(std::integral_constant<int, 4>{}, lse);
                else if (a.cols <= 1024) small(std::integral_constant<int, 16>{}, lse);
                else small(std::integral_constant<int, 32>{}, lse);
            };
            if (a.lse) sized(std::true_type{});
            else sized(std::false_type{});
            return;
        }
        for (int64_t row0 = 0; row0 < a.rows; row0 += a.run) {
            const int64_t rows = std::min(a.run, a.rows - row0);
            const unsigned blocks = (unsigned)rows;
            const dim3 tiles((unsigned)std::min(a.tiles, 4096), (unsigned)rows);
            auto both = [&](auto lse) {
                constexpr bool LSE = decltype(lse)::value;
                topk_groups_kernel<T, LSE><<<tiles, kTileGroups, 0, st>>>(a, row0);
                // (a workgroup of 1024 threads while they do not fill the compute units: bf16 [300, 50257], k = 200, 24.8 us with 256 and 29.8 with 1024, [200, 50257] 17.5 with them)
                if (for_a_wave<T>(rows, a.tiles, a.k)) topk_wave_kernel<T, LSE><<<(blocks + 3) / 4, kTileGroups, 0, st>>>(a, row0, rows);
                else topk_pick_kernel<T, LSE><<<blocks, rows <= 256 ? 1024 : 256, 0, st>>>(a, row0, rows);
            };
            if (a.lse) both(std::true_type{});
            else both(std::false_type{});
        }
    });
}

}  // namespace hpt
