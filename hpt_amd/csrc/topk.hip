// The k largest logits of each row, in order, and the log of the sum of exponentials of the row over a temperature.
//
// Two launches. The first reads the logits once, in tiles of 8192: each thread keeps the largest key of its 32 logits (and, where the sum is wanted, adds
// their exponentials below the tile's largest). The second has a workgroup for each row, which finds the first k places from those keys (top_rows.hpp).
// The first is bound by memory, the second by the latency of its steps.
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

int64_t rows_of_run(int64_t rows, size_t row_bytes) { return std::max<int64_t>(1, std::min<int64_t>(rows, (int64_t)(kMostRowScratch / row_bytes))); }
static int64_t tiles_of(int64_t cols) { return (cols + kTile - 1) / kTile; }
size_t topk_row_bytes(int dtype, int64_t cols, bool lse) {
    return (size_t)tiles_of(cols) * (kTileGroups * dtype_size(dtype) + (lse ? 2 * sizeof(double) : 0));
}

namespace {

template <class T, bool LSE>
__global__ __launch_bounds__(kTileGroups) void topk_groups_kernel(const TopkArgs a, int64_t row0, int64_t rows) {
    constexpr int VEC = 16 / sizeof(T), V = kTileVecs<T>;
    __shared__ uint32_t tops[4];
    __shared__ double sums[4];
    for (int64_t at = blockIdx.x; at < rows * a.tiles; at += gridDim.x) {
        const int64_t row = quotient(at, a.tiles);
        const int tile = (int)(at - row * a.tiles);
        Pack<T, VEC> p[V];
        load_tile<T>((const T*)a.x + offset_of(a.kept, row0 + row), tile, a.cols, p);
        const uint32_t key = most_key<T>(p);
        ((KeyOf<T>*)a.keys)[at * kTileGroups + threadIdx.x] = (KeyOf<T>)key;
        if constexpr (LSE) {
            const uint32_t top = block_reduce<MaxU>(key, tops);
            double add = 0.0;
            // (NaN, +inf and nothing but -inf are told from the largest alone)
            if (top < kInfKey<T> && top > kNegInfKey<T>) {
                const float most = value_of<T>(top);
                float part = 0.0f;
#pragma unroll
                for (int b = 0; b < V; ++b)
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        const float d = Elem<T>::widen(p[b].v[i]) - most;
                        part += __builtin_amdgcn_exp2f(fmaf(d, a.steps.hi, d * a.steps.lo));
                    }
                add = part;
            }
            add = block_reduce<SumD>(add, sums);
            if (threadIdx.x == 0) {
                a.sums[2 * at] = top >= kInfKey<T> || top <= kNegInfKey<T> ? (top == kInfKey<T> ? __builtin_huge_val() : top <= kNegInfKey<T> ? -__builtin_huge_val() : __builtin_nan("")) : (double)value_of<T>(top);
                a.sums[2 * at + 1] = add;
            }
        }
    }
}

template <class T, bool LSE>
__global__ __launch_bounds__(1024) void topk_pick_kernel(const TopkArgs a, int64_t row0, int64_t rows) {
    __shared__ TopShared s;
    __shared__ double place[16], place2[16];
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const int64_t row = row0 + r;
        const T* x = (const T*)a.x + offset_of(a.kept, row);
        if constexpr (LSE) {
            const double* p = a.sums + 2 * r * a.tiles;
            double top = -__builtin_huge_val(), nan = 0.0;
            for (int t = threadIdx.x; t < a.tiles; t += blockDim.x) {
                top = fmax(top, p[2 * t]);
                nan += p[2 * t] != p[2 * t] ? 1.0 : 0.0;
            }
            struct MaxD {
                __device__ static __forceinline__ double comb(double a, double b) { return fmax(a, b); }
            };
            top = block_reduce<MaxD>(top, place);
            double sum = 0.0;
            for (int t = threadIdx.x; t < a.tiles; t += blockDim.x)
                if (p[2 * t + 1] > 0.0) sum += p[2 * t + 1] * exp((p[2 * t] - top) * a.inv_temperature);
            sum = block_reduce<SumD>(sum, place2);
            nan = block_reduce<SumD>(nan, place);
            if (threadIdx.x == 0) {
                double lse = top * a.inv_temperature;
                if (nan > 0.0) lse = __builtin_nan("");
                else if (fabs(top) < __builtin_huge_val()) lse += log(sum);
                a.lse[row] = (float)lse;
            }
        }
        const int n = collect_top<T>(s, x, a.cols, (const KeyOf<T>*)a.keys + r * a.tiles * kTileGroups, a.tiles, a.k);
        rank_top(s, n, a.k, [&](int rank, uint64_t at) {
            const uint32_t i = index_of(at);
            ((T*)a.values)[row * a.k + rank] = x[i];
            if (a.index64) ((int64_t*)a.index)[row * a.k + rank] = i;
            else ((int32_t*)a.index)[row * a.k + rank] = (int32_t)i;
        });
        __syncthreads();
    }
}

}  // namespace

void launch_topk(int dtype, const TopkArgs& a, hipStream_t st) {
    HPT_WITH_TYPE(dtype, {
        for (int64_t row0 = 0; row0 < a.rows; row0 += a.run) {
            const int64_t rows = std::min(a.run, a.rows - row0);
            const unsigned tiles = (unsigned)std::min<int64_t>(rows * a.tiles, 1 << 20);
            // few rows: more threads for each
            const unsigned threads = rows <= 512 ? 1024 : 256;
            if (a.lse) {
                topk_groups_kernel<T, true><<<tiles, kTileGroups, 0, st>>>(a, row0, rows);
                topk_pick_kernel<T, true><<<(unsigned)std::min<int64_t>(rows, 1 << 20), threads, 0, st>>>(a, row0, rows);
            } else {
                topk_groups_kernel<T, false><<<tiles, kTileGroups, 0, st>>>(a, row0, rows);
                topk_pick_kernel<T, false><<<(unsigned)std::min<int64_t>(rows, 1 << 20), threads, 0, st>>>(a, row0, rows);
            }
        }
    });
}

}  // namespace hpt
