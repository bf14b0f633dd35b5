// The first k places of a row's order, from the largest key of each group of 32 neighbours: shared by topk.hip and the rows of sample.hip that
// are cut to few tokens. One workgroup for each row.
//
// The k-th largest of the groups' keys is at most the k-th largest logit's (each group's largest is one of the row's logits), and so is any key below it. One is found
// from a histogram of the distances below the row's largest, in sixteenths of a power of two; only groups that reach it are read again: k of them, and
// some more. What they hold at or above that key is collected, and its first k places are the row's. Where that is too much, the k-th place itself is found by sweeps
// over the row, eight bits of its key at a time, and the row is collected in its order: a row of few different values, and one whose first k logits lie on both sides of zero or next to it (their distances
// run through all powers of two down to it), or far from zero against their distances (a sixteenth of a power of two holds many of them). us of bf16 [4096, 50257], k = 64, whose first places lie between 6 and
// 15, and with -8 and -100 added: 102, 624 and 567; f32 [37, 50257], k = 33: 13, 120 and 92; as log-probabilities both are as fast as at first.
//
// Up to 64 places of very many rows are a wavefront's work, which waits for nobody (wave_top): its histogram is a search by halves over the largest of each vector of keys.
#pragma once

#include "vocab_rows.hpp"

namespace hpt {

// CAP: places collected.
template <int CAP> struct TopShared {
    uint64_t list[CAP];
    uint32_t groups[CAP];  // those that are read again
    uint16_t by_digit[CAP];
    Digits digits;
    uint32_t count, many, digit, above;
    uint32_t most, least;  // no collected key is above or below
    uint32_t waves[2 * 16];
};

// The k-th largest key of a row, eight bits at a time; `left`: how many of those that equal it are among the first k. sweep(f) calls f(key) for each.
template <int BITS, int CAP, class Sweep> __device__ __forceinline__ uint32_t kth_key(TopShared<CAP>& s, uint32_t k, uint32_t& left, Sweep&& sweep) {
    uint32_t prefix = 0;
#pragma clang loop unroll(disable)
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
    left = k;
    return prefix;
}

// The first k places by the row alone, in no order, into s.list.
template <class T, int CAP> __device__ __forceinline__ void collect_by_sweeps(TopShared<CAP>& s, const LogitRow<T>& row, int k) {
    constexpr int VEC = 16 / sizeof(T);
    uint32_t ties;
    const int vecs = row.vecs();
    const uint32_t key = kth_key<kKeyBits<T>>(s, k, ties, [&](auto&& f) {
        for (int v = threadIdx.x; v < vecs; v += blockDim.x) {
            const Pack<T, VEC> p = row.raw(v);
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (row.holds(v * VEC + i)) f(key_of(p.v[i]));
        }
    });
    // in the row's own order, so that of the equal ones the first are taken
    uint32_t over = 0, equal = 0;  // of both so far
#pragma clang loop unroll(disable)
    for (int v0 = 0; v0 < vecs; v0 += blockDim.x) {
        const int v = v0 + threadIdx.x;
        Pack<T, VEC> p;
        if (v < vecs) p = row.raw(v);
        uint32_t more = 0, same = 0;
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (row.holds(v * VEC + i)) {
                const uint32_t q = key_of(p.v[i]);
                more += q > key;
                same += q == key;
            }
        const uint32_t both = more | same << 16, sum = wave_scan(both);  // (at most 8 * 1024 of each)
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
                if (row.holds(v * VEC + i)) {
                    const uint32_t q = key_of(p.v[i]);
                    if (q > key) s.list[a++] = place_of(q, v * VEC + i - row.lead);  // (fewer than k)
                    else if (q == key) {
                        if (b < ties) s.list[k - ties + b] = place_of(q, v * VEC + i - row.lead);
                        ++b;
                    }
                }
        over += all & 0xFFFF;
        equal += all >> 16;
    }
    if (threadIdx.x == 0) s.least = key;
    __syncthreads();
}

// Collects into s.list (unordered) the first k places of the row and perhaps some behind them; returns how many. k <= cols, k <= CAP. Each tile's keys lie
// side by side, `apart` bytes from the next one's.
template <class T, int CAP> __device__ __forceinline__ int collect_top(TopShared<CAP>& s, const LogitRow<T>& row, const void* keys, int tiles, int k, size_t apart) {
    constexpr int VEC = 16 / sizeof(T), V = kTileVecs<T>;
    constexpr int KV = 16 / sizeof(KeyOf<T>), per = kTileGroups / KV;  // keys of a vector, vectors of a tile
    constexpr int SHIFT = (std::is_same<T, f16_t>::value ? 10 : std::is_same<T, float>::value ? 23 : 7) - 4;
    const int threads = (int)blockDim.x, vecs = tiles * per, rounds = (vecs + threads - 1) / threads;
    typedef Pack<KeyOf<T>, KV> Keys;
    auto keys_at = [&](int r) {
        const int i = r * threads + (int)threadIdx.x;
        Keys p;
        __builtin_memset(&p, 0, sizeof p);
        if (i < vecs) p = load_pack<KeyOf<T>, KV>((const KeyOf<T>*)((const char*)keys + (i / per) * apart) + (i % per) * KV);
        return p;
    };
    // (two vectors of a thread stay; keys of longer rows are fetched again)
    const Keys first = keys_at(0), second = rounds > 1 ? keys_at(1) : first;
    auto keys_of_round = [&](int r) { return r == 0 ? first : r == 1 ? second : keys_at(r); };
    uint32_t most = 0;
    for (int r = 0; r < rounds; ++r) {
        const Keys p = keys_of_round(r);
#pragma unroll
        for (int j = 0; j < KV; ++j) most = max(most, (uint32_t)p.v[j]);
    }
    s.digits.clear();
    if (threadIdx.x == 0) s.count = s.many = 0;
    most = wave_max(most);
    if ((threadIdx.x & 63) == 0) s.waves[threadIdx.x >> 6] = most;
    __syncthreads();
    most = wave_max((threadIdx.x & 63) < blockDim.x / 64 ? s.waves[threadIdx.x & 63] : 0);  // (every wavefront for itself)
    for (int r = 0; r < rounds; ++r) {
        const Keys p = keys_of_round(r);
#pragma unroll
        for (int j = 0; j < KV; ++j)
            if (p.v[j]) s.digits.add(255 - min((most - p.v[j]) >> SHIFT, 255u));
    }
    __syncthreads();
    if (threadIdx.x < 64) {
        uint32_t d, above;
        s.digits.find(k, d, above);
        if (threadIdx.x == 0) s.digit = d;
    }
    __syncthreads();
    // (the last of the distances holds all that is further)
    const uint32_t far = (256 - s.digit) << SHIFT, least = s.digit == 0 || far > most ? 1 : most - far + 1;
    for (int r = 0; r < rounds; ++r) {
        const Keys p = keys_of_round(r);
        uint32_t hits = 0;
#pragma unroll
        for (int j = 0; j < KV; ++j) hits |= p.v[j] >= least ? 1u << j : 0;
        while (hits) {
            const int j = __builtin_ctz(hits);
            hits &= hits - 1;
            const uint32_t at = atomicAdd(&s.many, 1u);
            if (at < CAP) s.groups[at] = (r * threads + threadIdx.x) * KV + j;
        }
    }
    __syncthreads();
    const int many = (int)s.many;
    if (threadIdx.x == 0) {
        s.most = most;
        s.least = least;
    }
    if (many <= CAP) {
        // N vectors of a thread on their way together
        auto look = [&](auto vectors) {
            constexpr int N = decltype(vectors)::value;
#pragma clang loop unroll(disable)
            for (int w0 = threadIdx.x; w0 < many * V; w0 += N * threads) {
                Pack<T, VEC> p[N];
                int first[N];
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    const int w = w0 + n * threads, v = group_vec<T>(s.groups[min(w / V, many - 1)], w % V);
                    first[n] = w < many * V ? v * VEC : row.end;
                    p[n] = row.raw(min(v, row.vecs() - 1));
                }
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    const int e = first[n];
                    if (e >= row.end) continue;
                    uint32_t key[VEC], hits = 0;
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        key[i] = key_of(p[n].v[i]);
                        hits |= key[i] >= least && row.holds(e + i) ? 1u << i : 0;
                    }
                    if (hits) {
                        uint32_t at = atomicAdd(&s.count, (uint32_t)__builtin_popcount(hits));
#pragma unroll
                        for (int i = 0; i < VEC; ++i)
                            if (hits >> i & 1) {
                                if (at < CAP) s.list[at] = place_of(key[i], e + i - row.lead);
                                ++at;
                            }
                    }
                }
            }
        };
        if (many * V <= threads) look(std::integral_constant<int, 1>{});
        else look(std::integral_constant<int, 4>{});
        __syncthreads();
        if (s.count <= CAP) return (int)s.count;
    }
    collect_by_sweeps<T>(s, row, k);
    return k;
}

// ---- a wavefront's form ---------------------------------------------------------------------------

constexpr int kWaveTop = 64;     // places at most
constexpr int kWaveList = 256;   // places, groups and vectors of keys that are collected
constexpr int kWaveRounds = 20;  // vectors of keys of a lane
struct WaveShared {
    union {
        uint32_t tops[kWaveRounds * 64];  // the largest of each vector of keys
        uint64_t list[kWaveList];
    };
    uint32_t vectors[kWaveList], groups[kWaveList];
};
// Whether rows are for it: fewer vectors of keys than places would find no bound, and it takes more rows than a workgroup each fills the compute units with. (us, a wavefront and a workgroup of 256, top-k:
// bf16 [300, 50257] k = 20 16.3 / 15.1, 64 24.3 / 18.0; [700, 50257] 23.5 / 23.0, 32.9 / 25.8; [2000, 50257] 42.5 / 49.0, 54.9 / 54.9, of 100 68 / 58; [4096, 50257] 84.7 / 105, 95.7 / 113.)
template <class T> __host__ __device__ constexpr bool for_a_wave(int64_t rows, int tiles, int k) {
    constexpr int per = kTileGroups * (int)sizeof(T) / 16;
    return rows > 1024 && k <= kWaveTop && tiles * per >= 2 * k && tiles * per <= kWaveRounds * 64;
}
__device__ __forceinline__ void wave_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }  // (a wavefront's accesses to LDS are in order)
__device__ __forceinline__ int lanes_before(uint64_t who) { return __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0)); }

// Collects into s.list (unordered) the first k places of the row and perhaps some behind them; returns how many, or -1 where that is too much.
template <class T> __device__ __forceinline__ int wave_top(WaveShared& s, const LogitRow<T>& row, const void* keys, int tiles, int k, size_t apart) {
    constexpr int VEC = 16 / sizeof(T), V = kTileVecs<T>;
    constexpr int KV = 16 / sizeof(KeyOf<T>), per = kTileGroups / KV;
    constexpr int SHIFT = (std::is_same<T, f16_t>::value ? 10 : std::is_same<T, float>::value ? 23 : 7) - 4;
    typedef Pack<KeyOf<T>, KV> Keys;
    const int lane = threadIdx.x & 63, vecs = tiles * per, rounds = (vecs + 63) / 64;
    auto keys_at = [&](int i) { return load_pack<KeyOf<T>, KV>((const KeyOf<T>*)((const char*)keys + (i / per) * apart) + (i % per) * KV); };
    // the largest of each vector of keys, four vectors on their way together
    uint32_t most = 0;
#pragma clang loop unroll(disable)
    for (int c = 0; c < rounds; c += 4) {
        Keys p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = keys_at(min((c + i) * 64 + lane, vecs - 1));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < KV; ++j) m = max(m, (uint32_t)p[i].v[j]);
            s.tops[(c + i) * 64 + lane] = (c + i) * 64 + lane < vecs ? m : 0;
            most = max(most, m);
        }
    }
    static_assert(kWaveRounds % 4 == 0, "the last round of four stays within");
    most = wave_max(most);
    // the smallest distance below the largest, in sixteenths of a power of two, that k of them are within
    auto from = [&](int d) {
        const uint32_t far = (uint32_t)(d + 1) << SHIFT;
        return d == 255 || far > most ? 1u : most - far + 1;
    };
    int lo = -1, hi = 255;
#pragma clang loop unroll(disable)
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        const uint32_t least = from(mid);
        int n = 0;
        for (int c = 0; c < rounds; ++c) n += __builtin_popcountll(__ballot(s.tops[c * 64 + lane] >= least));
        (n >= k ? hi : lo) = mid;
    }
    const uint32_t least = from(hi);
    int na = 0, nb = 0, n = 0;
    for (int c = 0; c < rounds; ++c) {
        const bool want = s.tops[c * 64 + lane] >= least;
        const uint64_t who = __ballot(want);
        const int at = na + lanes_before(who);
        if (want && at < kWaveList) s.vectors[at] = c * 64 + lane;
        na += __builtin_popcountll(who);
    }
    if (na > kWaveList) return -1;
    wave_fence();
#pragma clang loop unroll(disable)
    for (int i0 = 0; i0 < na; i0 += 64) {
        const uint32_t v = s.vectors[min(i0 + lane, na - 1)];
        const Keys p = keys_at(v);
        uint32_t hits = 0;
#pragma unroll
        for (int j = 0; j < KV; ++j) hits |= p.v[j] >= least ? 1u << j : 0;
        if (i0 + lane >= na) hits = 0;
        while (__any(hits)) {
            const uint64_t who = __ballot(hits != 0);
            const int at = nb + lanes_before(who);
            if (hits) {
                if (at < kWaveList) s.groups[at] = v * KV + __builtin_ctz(hits);
                hits &= hits - 1;
            }
            nb += __builtin_popcountll(who);
        }
    }
    if (nb > kWaveList) return -1;
    wave_fence();
#pragma clang loop unroll(disable)
    for (int w0 = 0; w0 < nb * V; w0 += 64 * 4) {
        Pack<T, VEC> p[4];
        int e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int w = w0 + i * 64 + lane;
            const int v = group_vec<T>(s.groups[min(w / V, nb - 1)], w % V);
            e[i] = w < nb * V ? v * VEC : row.end;
            p[i] = row.raw(min(v, row.vecs() - 1));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (w0 + i * 64 >= nb * V) continue;
            uint32_t key[VEC], hits = 0;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                key[j] = key_of(p[i].v[j]);
                hits |= key[j] >= least && row.holds(e[i] + j) ? 1u << j : 0;
            }
            const int mine = __builtin_popcount(hits);
            const int upto = wave_scan(mine);
            int at = n + upto - mine;
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (hits >> j & 1) {
                    if (at < kWaveList) s.list[at] = place_of(key[j], e[i] + j - row.lead);
                    ++at;
                }
            n += lane_of(upto, 63);
        }
    }
    wave_fence();
    return n <= kWaveList ? n : -1;
}

// Gives each of the first k of `n` places that a wavefront has collected to `out(rank, place)`.
template <class Out> __device__ __forceinline__ void wave_rank(const WaveShared& s, int n, int k, Out&& out) {
    for (int i = threadIdx.x & 63; i < n; i += 64) {
        const uint64_t mine = s.list[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) rank += s.list[j] > mine;
        if (rank < k) out(rank, mine);
    }
}

// Gives each of the first k of `n` collected places to `out(rank, place)`, the ranks counted from 0. Up to kMostRanked of them a thread counts what is before its own. Of more it
// counts only those of its own digit: eight bits below the largest key, which deal them out first. They are sorted where one digit has too many (keys that are equal).
constexpr int kMostRanked = 128, kMostOfDigit = 256;
template <int CAP, class Out> __device__ __forceinline__ void rank_top(TopShared<CAP>& s, int n, int k, Out&& out) {
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
    uint32_t *upto = s.digits.n, *from = upto + 256;  // where a digit's places end (so far) and begin
    const uint32_t most = s.most, width = most - s.least, shift = width < 256 ? 0 : 24 - __builtin_clz(width);
    auto digit = [&](uint64_t place) { return min((most - key_of_place(place)) >> shift, 255u); };
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += blockDim.x) upto[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x) atomicAdd(&upto[digit(s.list[i])], 1u);
    __syncthreads();
    if (threadIdx.x < 64) {
        uint32_t c[4], sum = 0, largest = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            c[i] = upto[threadIdx.x * 4 + i];
            sum += c[i];
            largest = max(largest, c[i]);
        }
        largest = wave_max(largest);
        uint32_t at = wave_scan(sum) - sum;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            upto[threadIdx.x * 4 + i] = from[threadIdx.x * 4 + i] = at;
            at += c[i];
        }
        if (threadIdx.x == 0) s.many = largest;
    }
    __syncthreads();
    if (s.many <= kMostOfDigit) {
        for (int i = threadIdx.x; i < n; i += blockDim.x) s.by_digit[atomicAdd(&upto[digit(s.list[i])], 1u)] = (uint16_t)i;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += blockDim.x) {
            const uint64_t mine = s.list[i];
            const uint32_t d = digit(mine), end = upto[d];
            uint32_t rank = from[d];
            if (rank >= (uint32_t)k) continue;
#pragma unroll 4
            for (uint32_t j = rank, all = end; j < all; ++j) rank += s.list[s.by_digit[j]] > mine;
            if (rank < (uint32_t)k) out(rank, mine);
        }
        return;
    }
    int size = 256;
    while (size < n) size <<= 1;
    for (int i = n + threadIdx.x; i < size; i += blockDim.x) s.list[i] = 0;
    sort_places(s.list, size);
    for (int i = threadIdx.x; i < k; i += blockDim.x) out(i, s.list[i]);
}

}  // namespace hpt
