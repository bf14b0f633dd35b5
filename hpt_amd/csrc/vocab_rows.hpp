// Device-side pieces that the operators over rows of logits share (topk.hip, sample.hip, distill_loss.hip): logits as order keys, a tile of
// a row in a workgroup's registers, and the search for a place in a row's order.
//
// The order of a row's logits: NaN before everything, then the larger value, equal ones (and -0, +0) by their index. A key orders as the
// value does, 0 is below all keys; a place is a key with the index behind it, counted down, so that places of a row differ.
#pragma once

#include "block_rows.hpp"

namespace hpt {

template <class T> struct Bits {
    using type = uint16_t;
    static constexpr uint32_t sign = 0x8000u, all = 0xFFFFu, inf = std::is_same<T, f16_t>::value ? 0x7C00u : 0x7F80u;
};
template <> struct Bits<float> {
    using type = uint32_t;
    static constexpr uint32_t sign = 0x80000000u, all = 0xFFFFFFFFu, inf = 0x7F800000u;
};
template <class T> using KeyOf = typename Bits<T>::type;
template <class T> constexpr uint32_t kNanKey = Bits<T>::all;
template <class T> constexpr uint32_t kInfKey = Bits<T>::sign | Bits<T>::inf;
template <class T> constexpr uint32_t kNegInfKey = ~(Bits<T>::sign | Bits<T>::inf) & Bits<T>::all;
template <class T> constexpr int kKeyBits = 8 * sizeof(T);

template <class T> __device__ __forceinline__ uint32_t bits_of(T x) { return __builtin_bit_cast(KeyOf<T>, x); }
template <class T> __device__ __forceinline__ uint32_t key_of_bits(uint32_t b) {
    using B = Bits<T>;
    if ((b & ~B::sign) > B::inf) return kNanKey<T>;
    if (b == B::sign) b = 0;
    return b & B::sign ? ~b & B::all : b | B::sign;
}
template <class T> __device__ __forceinline__ uint32_t key_of(T x) { return key_of_bits<T>(bits_of(x)); }
// The value of a key that is no NaN's.
template <class T> __device__ __forceinline__ float value_of(uint32_t key) {
    using B = Bits<T>;
    const uint32_t b = key & B::sign ? key & ~B::sign : ~key & B::all;
    return Elem<T>::widen(__builtin_bit_cast(T, (KeyOf<T>)b));
}

// The largest key of a vector: two-byte logits two at a time, as signed numbers whose order is the values'. Negative NaNs, which that order puts below
// everything, show as the largest plain bits.
template <class T> __device__ __forceinline__ uint32_t most_key(const Pack<T, 16 / sizeof(T)>& p) {
    using B = Bits<T>;
    typedef int16_t s16x2 __attribute__((ext_vector_type(2)));
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    if constexpr (sizeof(T) == 2) {
        s16x2 top = {-32768, -32768};
        u16x2 raw = {0, 0};
        struct Words {
            uint32_t w[4];
        };
        const Words words = __builtin_bit_cast(Words, p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const s16x2 s = __builtin_bit_cast(s16x2, words.w[i]);
            const s16x2 o = s ^ ((s >> 15) & (int16_t)0x7FFF);
            top = __builtin_elementwise_max(top, o);
            raw = __builtin_elementwise_max(raw, __builtin_bit_cast(u16x2, words.w[i]));
        }
        const int16_t t = top.x > top.y ? top.x : top.y;
        const uint16_t r = raw.x > raw.y ? raw.x : raw.y;
        if (r > (B::sign | B::inf)) return kNanKey<T>;
        return key_of_bits<T>((uint16_t)(t ^ ((t >> 15) & 0x7FFF)));
    } else {
        int32_t top = INT32_MIN;
        uint32_t raw = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t u = bits_of(p.v[i]);
            const int32_t s = (int32_t)u, o = s ^ ((s >> 31) & 0x7FFFFFFF);
            top = top > o ? top : o;
            raw = raw > u ? raw : u;
        }
        if (raw > (B::sign | B::inf)) return kNanKey<T>;
        return key_of_bits<T>((uint32_t)(top ^ ((top >> 31) & 0x7FFFFFFF)));
    }
}

// A row of logits as the aligned vectors that contain it: `lead` elements before its first one (they may be another row's) and those behind its last are -inf. (Unaligned
// vectors, from the row's start on: loss of distillation alone, bf16 [8192, 50257] 206 -> 179 us.)
template <class T> struct LogitRow {
    static constexpr int VEC = 16 / sizeof(T);
    const T* base;
    int lead, end;  // the row is at lead ... end - 1
    __device__ __forceinline__ LogitRow(const T* x, int cols) : lead((int)((uintptr_t)x & 15) / (int)sizeof(T)), end(lead + cols) { base = x - lead; }
    __device__ __forceinline__ bool holds(int e) const { return e >= lead && e < end; }
    __device__ __forceinline__ int vecs() const { return (end + VEC - 1) / VEC; }
    // v below vecs()
    __device__ __forceinline__ Pack<T, VEC> raw(int v) const { return load_pack<T, VEC>(base + (int64_t)v * VEC); }
    __device__ __forceinline__ void clean(Pack<T, VEC>& p, int v) const {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (!holds(v * VEC + i)) p.v[i] = Elem<T>::narrow(-__builtin_huge_valf());
    }
};
// Vector b of the 32 logits that a thread has of a tile: a wavefront has 2048 neighbours, and its vectors lie lane beside lane.
template <class T> constexpr int kTileVecs = kTile * sizeof(T) / 16 / kTileGroups;  // of a thread
template <class T> __device__ __forceinline__ int tile_vec(int tile, int b, int thread) {
    return (tile * (kTileGroups / 64) + (thread >> 6)) * (64 * kTileVecs<T>) + b * 64 + (thread & 63);
}
// All of them: their loads are on their way together, and only a tile with an end of the row looks for it.
template <class T> __device__ __forceinline__ void load_tile(const LogitRow<T>& row, int tile, Pack<T, 16 / sizeof(T)> (&p)[kTileVecs<T>]) {
    constexpr int VEC = 16 / sizeof(T);
    if ((tile == 0 && row.lead) || (tile + 1) * (int64_t)kTile > row.end) {
        const int last = row.vecs() - 1;
#pragma unroll
        for (int b = 0; b < kTileVecs<T>; ++b) p[b] = row.raw(min(tile_vec<T>(tile, b, threadIdx.x), last));
#pragma unroll
        for (int b = 0; b < kTileVecs<T>; ++b) row.clean(p[b], tile_vec<T>(tile, b, threadIdx.x));
    } else {
        const T* at = row.base + (int64_t)tile_vec<T>(tile, 0, threadIdx.x) * VEC;
#pragma unroll
        for (int b = 0; b < kTileVecs<T>; ++b) p[b] = load_pack<T, VEC>(at + b * 64 * VEC);
    }
}

// A tile's logits are dealt to groups of 32 neighbours, whose largest keys its threads get one each: lane l that of the kTileVecs vectors of its wavefront from
// (l % kTileVecs) * 64 + l / kTileVecs * kTileVecs on (vectors that neighbouring lanes have loaded together; 64 or 128 bytes side by side, so that a group that is read again is one or two lines).
// Each of 4 (8) lanes gives away half of its vectors' largest for the other half of its partner's, then half of those, until one is left.
template <class A, int N, class Comb> __device__ __forceinline__ A trade(A (&m)[N], Comb&& comb) {
    const int lane = threadIdx.x & 63;
    if constexpr (N == 8) {
        const bool upper = lane & 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const A give = upper ? m[i] : m[i + 4], keep = upper ? m[i + 4] : m[i];
            m[i] = comb(keep, dpp_move<0x141>(give));  // (mirrored within eight)
        }
    }
    {
        const bool upper = lane & 2;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const A give = upper ? m[i] : m[i + 2], keep = upper ? m[i + 2] : m[i];
            m[i] = comb(keep, dpp_move<0x4E>(give));
        }
    }
    const bool upper = lane & 1;
    const A give = upper ? m[0] : m[1], keep = upper ? m[1] : m[0];
    return comb(keep, dpp_move<0xB1>(give));
}
template <class T> __device__ __forceinline__ uint32_t group_key(const Pack<T, 16 / sizeof(T)> (&p)[kTileVecs<T>]) {
    using B = Bits<T>;
    constexpr int V = kTileVecs<T>;
    uint32_t m[V];
    if constexpr (sizeof(T) == 2) {
        // two by two, as signed numbers that order as the values do, and the lanes' halves met last; but negative NaNs, which show as the largest plain bits, take the way of single logits
        typedef int16_t s16x2 __attribute__((ext_vector_type(2)));
        typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
        u16x2 raw = {0, 0};
#pragma unroll
        for (int b = 0; b < V; ++b) {
            struct Words {
                uint32_t w[4];
            };
            const Words words = __builtin_bit_cast(Words, p[b]);
            s16x2 top = {-32768, -32768};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const s16x2 s = __builtin_bit_cast(s16x2, words.w[i]);
                top = __builtin_elementwise_max(top, s ^ ((s >> 15) & (int16_t)0x7FFF));
                raw = __builtin_elementwise_max(raw, __builtin_bit_cast(u16x2, words.w[i]));
            }
            m[b] = __builtin_bit_cast(uint32_t, top);
        }
        if (!__any(max((uint32_t)raw.x, (uint32_t)raw.y) > (B::sign | B::inf))) {
            const s16x2 top = __builtin_bit_cast(s16x2, trade(m, [](uint32_t a, uint32_t b) {
                return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(s16x2, a), __builtin_bit_cast(s16x2, b)));
            }));
            const uint32_t key = (uint16_t)(top.x > top.y ? top.x : top.y) ^ B::sign;
            return key > kInfKey<T> ? kNanKey<T> : key == B::sign - 1 ? B::sign : key;  // (-0 is 0)
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) m[i] = most_key<T>(p[i]);
    return trade(m, [](uint32_t a, uint32_t b) { return max(a, b); });
}
// Vector w of the group with number g of a row.
template <class T> __device__ __forceinline__ int group_vec(uint32_t g, int w) {
    constexpr int V = kTileVecs<T>;
    const int l = g % 64;
    return g / 64 * (64 * V) + l % V * 64 + l / V * V + w;
}
// v of lane l, the same l for all lanes, and of the lane before this one (0 for lane 0). By the vector unit alone, as the scan below is: through LDS each of their
// steps would wait some 130 cycles, which a workgroup that has a row for itself cannot fill. Whole wavefronts only.
template <class A> __device__ __forceinline__ A lane_of(A v, int l) {
    union {
        A a;
        int w[sizeof(A) / 4];
    } in, out;
    in.a = v;
    l = __builtin_amdgcn_readfirstlane(l);
#pragma unroll
    for (int i = 0; i < (int)sizeof(A) / 4; ++i) out.w[i] = __builtin_amdgcn_readlane(in.w[i], l);
    return out.a;
}
// (along a DPP pattern, 0 where it has nothing to give or ROWS, a bit for each 16 lanes, leaves a lane out)
template <int CTRL, int ROWS, class A> __device__ __forceinline__ A dpp_or_zero(A v) {
    union {
        A a;
        int w[sizeof(A) / 4];
    } in, out;
    in.a = v;
#pragma unroll
    for (int i = 0; i < (int)sizeof(A) / 4; ++i) out.w[i] = __builtin_amdgcn_update_dpp(0, in.w[i], CTRL, ROWS, 0xF, true);
    return out.a;
}
template <class A> __device__ __forceinline__ A lane_before(A v) { return dpp_or_zero<0x138, 0xF>(v); }  // wave_shr:1
// The sum of v over this lane and those before it: within 16 lanes by shifts of 1, 2, 4, 8, then the last of a row added to the next one, and of the first two to the last two.
template <class A> __device__ __forceinline__ A wave_scan(A v) {
    v += dpp_or_zero<0x111, 0xF>(v);
    v += dpp_or_zero<0x112, 0xF>(v);
    v += dpp_or_zero<0x114, 0xF>(v);
    v += dpp_or_zero<0x118, 0xF>(v);
    v += dpp_or_zero<0x142, 0xA>(v);  // row_bcast:15
    v += dpp_or_zero<0x143, 0xC>(v);  // row_bcast:31
    return v;
}
// The largest of a wavefront's, in the same way.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = max(v, dpp_or_zero<0x111, 0xF>(v));
    v = max(v, dpp_or_zero<0x112, 0xF>(v));
    v = max(v, dpp_or_zero<0x114, 0xF>(v));
    v = max(v, dpp_or_zero<0x118, 0xF>(v));
    v = max(v, dpp_or_zero<0x142, 0xA>(v));
    v = max(v, dpp_or_zero<0x143, 0xC>(v));
    return lane_of(v, 63);
}
// The sum of N numbers (a power of two) of this lane, two by two: log2 N roundings deep.
template <int N> __device__ __forceinline__ float sum_by_twos(float (&v)[N]) {
#pragma unroll
    for (int w = N / 2; w > 0; w /= 2)
#pragma unroll
        for (int i = 0; i < w; ++i) v[i] += v[i + w];
    return v[0];
}
// The sum of v over the threads before this one; `total`: over all of them. Every order is fixed. `place`: one number for each wavefront.
__device__ __forceinline__ double scan_before(double v, double* place, double& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const double sum = wave_scan(v);
    __syncthreads();
    if (lane == 63) place[wave] = sum;
    __syncthreads();
    // (every wavefront adds them up for itself, a lane each)
    const double upto = wave_scan(lane < waves ? place[lane] : 0.0), shifted = lane_before(sum);
    total = lane_of(upto, 63);
    const double before = lane_of(upto, max(wave - 1, 0));
    return (wave ? before : 0.0) + shifted;
}

// Digits of eight bits: how many of what is looked at have each, in four tables that neighbouring lanes take in turn (the largest of a row's groups of logits
// have nearly all the same first digit, and lanes that add to one address wait for each other).
struct Digits {
    alignas(16) uint32_t n[256 * 4];
    __device__ __forceinline__ void clear() {
        for (int i = threadIdx.x; i < 256 * 4; i += blockDim.x) n[i] = 0;
    }
    __device__ __forceinline__ void add(uint32_t digit) { atomicAdd(&n[digit * 4 + (threadIdx.x & 3)], 1u); }
    // The digit of the k-th from the top (k >= 1), and how many have a larger one: called by the whole first wavefront after a barrier; 0 with all of them before it where there are fewer than k.
    __device__ __forceinline__ void find(uint32_t k, uint32_t& digit, uint32_t& above) const {
        const int lane = threadIdx.x & 63;
        uint32_t c[4], sum = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // (lane 0 has the four largest digits)
            const uint32_t* p = n + (255 - (lane * 4 + i)) * 4;
            c[i] = p[0] + p[1] + p[2] + p[3];
            sum += c[i];
        }
        const uint32_t upto = wave_scan(sum);
        const uint64_t reach = __ballot(upto >= k);
        const int at = reach ? __builtin_ctzll(reach) : 63;
        uint32_t before = upto - sum, d = 255 - lane * 4;
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (before + c[i] < k && d == (uint32_t)(255 - (lane * 4 + i))) {
                before += c[i];
                --d;
            }
        digit = lane_of(d, at);
        above = lane_of(before, at);
    }
};

// A place of the order in 64 bits.
__device__ __forceinline__ uint64_t place_of(uint32_t key, uint32_t index) { return ((uint64_t)key << 32) | (0xFFFFFFFFu - index); }
__device__ __forceinline__ uint32_t index_of(uint64_t place) { return 0xFFFFFFFFu - (uint32_t)place; }
__device__ __forceinline__ uint32_t key_of_place(uint64_t place) { return (uint32_t)(place >> 32); }

// Largest first; n a power of two, every thread of the workgroup. Steps within 128 neighbours stay with a wavefront, whose accesses to LDS are in order.
__device__ __forceinline__ void sort_places(uint64_t* list, int n) {
    __syncthreads();
    for (int size = 2; size <= n; size <<= 1)
        for (int stride = size >> 1; stride > 0; stride >>= 1) {
            for (int p = threadIdx.x; p < n / 2; p += blockDim.x) {
                const int i = 2 * p - (p & (stride - 1)), j = i + stride;
                const uint64_t a = list[i], b = list[j];
                if (((i & size) == 0) == (a < b)) {
                    list[i] = b;
                    list[j] = a;
                }
            }
            if (stride > 64 || (stride == 1 && size >= 128)) __syncthreads();
            else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    __syncthreads();
}

}  // namespace hpt
