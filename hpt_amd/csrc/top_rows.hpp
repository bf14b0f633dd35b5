// The first k places of a row's order, from the largest key of each thread's 32 logits: shared by topk.hip and the rows of sample.hip that
// are cut to few tokens. One workgroup for each row.
//
// The k-th largest of the groups' keys is at most the k-th largest logit's (each group's largest is one of the row's logits), so only groups that
// reach it are read again: k of them and those that tie. What they hold at or above that key is collected, and its first k places are the row's.
// Where that is too much (a row of few different values), the k-th place itself is found by sweeps over the row, eight bits of its key at a
// time, and the row is collected in its order.
#pragma once

#include "vocab_rows.hpp"

namespace hpt {

constexpr int kMostList = 2048;  // places collected
static_assert(kMostTop <= kMostList, "the first k fit the list");

struct TopShared {
    uint64_t list[kMostList];
    uint32_t groups[kMostList];  // those that are read again
    Digits digits;
    uint32_t count, many, digit, above;
    uint32_t waves[2 * 16];
};

// The k-th largest of `n` keys (0 where there are fewer), eight bits at a time; `each` gives the keys to a function: sweep(f) calls f(key) or passes.
template <int BITS, class Sweep> __device__ __forceinline__ uint32_t kth_key(TopShared& s, uint32_t k, uint32_t* left, Sweep&& sweep) {
    uint32_t prefix = 0;
    for (int shift = BITS - 8; shift >= 0; shift -= 8) {
        __syncthreads();
        s.digits.clear();
        __syncthreads();
        sweep([&](uint32_t key) {
            if (shift == BITS - 8 || key >> (shift + 8) == prefix >> (shift + 8)) s.digits.add((key >> shift) & 255);
        });
        __syncthreads();
        if (threadIdx.x < 64) {
            uint32_t d, above;
            s.digits.find(k, d, above);
            if (threadIdx.x == 0) {
                s.digit = d;
                s.above = above;
            }
        }
        __syncthreads();
        prefix |= s.digit << shift;
        k = k > s.above ? k - s.above : 1;
    }
    if (left) *left = k;  // so many of those that equal it
    return prefix;
}

// Collects into s.list (unordered) the first k <= kMostTop places of the row and perhaps some behind them; returns how many. k <= cols.
// Each tile's keys lie side by side, `apart` bytes from the next one's.
template <class T> __device__ __forceinline__ int collect_top(TopShared& s, const T* x, int cols, const void* keys, int tiles, int k, size_t apart = kTileGroups * sizeof(T)) {
    constexpr int VEC = 16 / sizeof(T), V = kTileVecs<T>;
    constexpr int KV = 16 / sizeof(KeyOf<T>);  // keys of a vector
    const int groups = tiles * kTileGroups;
    constexpr int per = kTileGroups / KV;
    auto keys_at = [&](int i) { return load_pack<KeyOf<T>, KV>((const KeyOf<T>*)((const char*)keys + (i / per) * apart) + (i % per) * KV); };
    const uint32_t least = kth_key<kKeyBits<T>>(s, k, nullptr, [&](auto&& f) {
        for (int i = threadIdx.x; i < groups / KV; i += blockDim.x) {
            const Pack<KeyOf<T>, KV> p = keys_at(i);
#pragma unroll
            for (int j = 0; j < KV; ++j) f((uint32_t)p.v[j]);
        }
    });
    __syncthreads();
    if (threadIdx.x == 0) s.count = s.many = 0;
    __syncthreads();
    const int rounds = (groups / KV + (int)blockDim.x - 1) / (int)blockDim.x;
    for (int r = 0; r < rounds; ++r) {
        const int i = r * (int)blockDim.x + (int)threadIdx.x;
        Pack<KeyOf<T>, KV> p;
        __builtin_memset(&p, 0, sizeof p);
        if (i < groups / KV) p = keys_at(i);
#pragma unroll
        for (int j = 0; j < KV; ++j) {
            const bool want = i < groups / KV && p.v[j] >= least;
            if (__any(want)) {
                const uint32_t at = reserve(want, &s.many);
                if (want && at < kMostList) s.groups[at] = i * KV + j;
            }
        }
    }
    __syncthreads();
    const int many = (int)s.many;
    if (many <= kMostList) {
        for (int w0 = 0; w0 < many * V; w0 += blockDim.x) {
            const int w = w0 + threadIdx.x;
            const bool on = w < many * V;
            Pack<T, VEC> p;
            int e = cols;
            if (on) {
                const uint32_t g = s.groups[w / V];
                const int v = tile_vec<T>(g / kTileGroups, w % V, g % kTileGroups);
                e = v * VEC;
                if (e < cols) p = logit_vec<T>(x, v, cols);
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const uint32_t key = e + i < cols ? key_of(p.v[i]) : 0;
                const bool want = e + i < cols && key >= least;
                if (__any(want)) {
                    const uint32_t at = reserve(want, &s.count);
                    if (want && at < kMostList) s.list[at] = place_of(key, e + i);
                }
            }
        }
        __syncthreads();
        if (s.count <= kMostList) return (int)s.count;
    }
    // the key of the k-th place, and how many of those that equal it belong to the first k
    uint32_t ties;
    const int vecs = (cols + VEC - 1) / VEC;
    const uint32_t key = kth_key<kKeyBits<T>>(s, k, &ties, [&](auto&& f) {
        for (int v = threadIdx.x; v < vecs; v += blockDim.x) {
            const Pack<T, VEC> p = logit_vec<T>(x, v, cols);
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (v * VEC + i < cols) f(key_of(p.v[i]));
        }
    });
    // in the row's own order, so that of the equal ones the first are taken
    uint32_t over = 0, equal = 0;  // of both so far
    for (int v0 = 0; v0 < vecs; v0 += blockDim.x) {
        const int v = v0 + threadIdx.x;
        Pack<T, VEC> p;
        if (v < vecs) p = logit_vec<T>(x, v, cols);
        uint32_t more = 0, same = 0;
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (v * VEC + i < cols) {
                const uint32_t q = key_of(p.v[i]);
                more += q > key;
                same += q == key;
            }
        uint32_t both = more | same << 16, sum = both;  // (at most 8 * 1024 of each)
#pragma unroll
        for (int w = 1; w < 64; w <<= 1) {
            const uint32_t o = __shfl_up(sum, w, 64);
            if ((int)(threadIdx.x & 63) >= w) sum += o;
        }
        __syncthreads();
        if ((threadIdx.x & 63) == 63) s.waves[threadIdx.x >> 6] = sum;
        __syncthreads();
        uint32_t before = sum - both, all = 0;
        for (int w = 0; w < (int)(blockDim.x >> 6); ++w) {
            if (w < (int)(threadIdx.x >> 6)) before += s.waves[w];
            all += s.waves[w];
        }
        uint32_t a = over + (before & 0xFFFF), b = equal + (before >> 16);
        if (v < vecs)
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (v * VEC + i < cols) {
                    const uint32_t q = key_of(p.v[i]);
                    if (q > key) s.list[a++] = place_of(q, v * VEC + i);  // (fewer than k)
                    else if (q == key) {
                        if (b < ties) s.list[k - ties + b] = place_of(q, v * VEC + i);
                        ++b;
                    }
                }
        over += all & 0xFFFF;
        equal += all >> 16;
    }
    __syncthreads();
    return k;
}

// Gives each of the first k of `n` collected places to `out(rank, place)`, the ranks counted from 0. Up to kMostRanked of them a thread counts what is before its own; beyond they are sorted.
constexpr int kMostRanked = 512;
template <class Out> __device__ __forceinline__ void rank_top(TopShared& s, int n, int k, Out&& out) {
    if (n <= kMostRanked) {
        for (int i = threadIdx.x; i < n; i += blockDim.x) {
            const uint64_t mine = s.list[i];
            int rank = 0;
#pragma unroll 8
            for (int j = 0; j < n; ++j) rank += s.list[j] > mine;
            if (rank < k) out(rank, mine);
        }
        return;
    }
    int size = 1024;
    while (size < n) size <<= 1;
    for (int i = n + threadIdx.x; i < size; i += blockDim.x) s.list[i] = 0;
    sort_places(s.list, size);
    for (int i = threadIdx.x; i < k; i += blockDim.x) out(i, s.list[i]);
}

}  // namespace hpt
