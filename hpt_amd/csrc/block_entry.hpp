// Operators around a transformer's blocks: what the C ABI hands to their launchers (rms_norm.hip, softmax_bias.hip,
// policy_loss.hip). The host has checked shapes, dtypes and overlaps; every tensor but `x` is contiguous.
#pragma once

#include <hip/hip_runtime_api.h>

#include "common.hpp"

namespace hpt {

// How a row of `cols` elements, taken as vectors of 16 bytes, is dealt to threads that keep it in registers: `tpr` of them share a
// row with `nc` vectors each. Up to a wavefront tpr is a power of two and a workgroup of 256 holds several rows; above, tpr is
// the workgroup, any number of wavefronts.
struct RowDeal {
    int tpr = 64;
    int nc = 1;
    int threads = 256;
    int rows_per_block() const { return threads / tpr; }
    bool held() const { return nc != 0; }  // otherwise the row does not fit: the streaming form
};

// `most`: vectors per thread that a kernel has registers for; `aim`: how many it should rather have; `least`: lanes a row has at least.
inline RowDeal deal_row(int64_t cols, size_t elem_size, int aim, int most, int least = 1) {
    const int64_t vecs = (cols * (int64_t)elem_size + 15) / 16;
    RowDeal d;
    if (vecs > (int64_t)most * 1024) {
        d.nc = 0;
        d.tpr = d.threads = 1024;
        return d;
    }
    int64_t t = (vecs + aim - 1) / aim;
    if (t <= 64) {
        d.tpr = least;
        while (d.tpr < t) d.tpr <<= 1;
        d.threads = 256;
    } else {
        d.tpr = d.threads = (int)(t + 63 > 1024 ? 1024 : (t + 63) / 64 * 64);
    }
    d.nc = (int)((vecs + d.tpr - 1) / d.tpr);
    return d;
}

// ---- RMS norm -----------------------------------------------------------------------------------

enum { QUANT_NONE = 0, QUANT_I8 = 1, QUANT_E4M3 = 2 };

struct RmsArgs {
    const void* x;      // rows of `cols` neighbouring elements
    Dims kept;          // where they start
    const void* res;    // or null
    const void* gamma;  // or null
    void* sum;          // x + res, or null
    void* out;
    float* scale;       // 8-bit outputs: rows x (cols / group)
    int64_t rows;
    int cols;
    int group;          // elements that share a scale
    float eps;
    int tpr;            // threads per row
};

void launch_rms_norm(int dtype, int quant, const RmsArgs& a, hipStream_t st);

struct RmsGradArgs {
    const void* x;
    Dims kept;
    const void* gy;     // the gradient of the norm's output
    const void* gsum;   // what else arrives at x, or null
    const void* gamma;  // or null
    void* gx;
    float* ggamma;      // or null
    float* partial;     // [blocks, cols]
    int64_t rows;
    int cols;
    float eps;
    int tpr;
};

// The rows of partial sums of gamma's gradient (0: none are needed).
int64_t rms_grad_partials(int dtype, int64_t rows, int64_t cols);
void launch_rms_norm_backward(int dtype, const RmsGradArgs& a, hipStream_t st);

// ---- softmax with a bucketed position bias --------------------------------------------------------

constexpr int kMostBuckets = 256;       // of both directions together
constexpr int kMostDistance = 4096;     // at which the last bucket may begin at the latest

// The buckets of key - query as distances. Bucket k of a direction holds the distances begin[k] ... begin[k + 1] - 1, its last
// one everything from begin[n - 1] on; `both`: keys behind the query take the buckets from n on.
struct Buckets {
    int n = 0;
    int both = 0;
    int far = 0;  // begin[n - 1]
    alignas(16) uint16_t begin[kMostBuckets] = {};  // from n on larger than any distance
};

// Throws where no such buckets exist.
Buckets make_buckets(int64_t total, bool both, int64_t max_distance);

struct BiasArgs {
    const void* x;        // [batch, heads, queries, keys], keys side by side
    Dims matrices;        // where each head's rows start
    int64_t query_stride;
    const void* table;    // [buckets, heads]
    int64_t table_bucket, table_head;  // its strides
    void* out;
    float* partial;       // split rows: (maximum, sum) of each part
    const void* lengths;  // [batch] of i32 or i64, or null
    int lengths64;
    int causal;
    int64_t heads, queries;
    int64_t rows;         // batch * heads * queries
    int keys;
    int64_t offset;       // position of the first query
    float scale;
    Buckets buckets;
    int tpr;
    int per_item;         // rows of one matrix that a workgroup takes
    int64_t chunks, items;  // such items: of a matrix, of all
    int split;            // > 1: workgroups that share a row
};

// Parts that a row is split into where there is scratch for it (1: none).
int bias_split(int dtype, int64_t rows, int64_t keys);
void launch_softmax_bias(int dtype, const BiasArgs& a, hipStream_t st);

struct BiasGradArgs {
    const void* p;
    const void* g;
    void* out;
    float* table_grad;    // [buckets, heads]
    float* partial;       // [items, buckets]
    const void* lengths;
    int lengths64;
    int causal;
    int64_t heads, queries, rows;
    int keys;
    int64_t offset;
    float scale;
    Buckets buckets;
    int tpr;
    int per_item;
    int64_t chunks, items;
};

// Rows of one matrix that a workgroup takes, and the number of such items.
int64_t bias_grad_items(int dtype, int64_t matrices, int64_t queries, int64_t keys, int* per_item);
void launch_softmax_bias_backward(int dtype, const BiasGradArgs& a, hipStream_t st);

// ---- policy loss ----------------------------------------------------------------------------------

struct PolicyArgs {
    const void* x;        // rows of `cols` neighbouring logits
    Dims kept;
    const void* token;    // [rows] of i32 or i64
    int token64;
    const float* old_logp;    // null: the log-probabilities alone
    const float* advantage;
    const float* reference;   // or null
    const void* mask;         // [rows] of f32 or bool, or null
    int mask_bool;
    double clip_low, clip_high, kl_weight;
    float *loss, *logp, *lse, *weight;
    double* each;         // [rows, 2] scratch of rows that are not split: the tokens' losses and slopes, times the mask
    double* partial;      // [rows, split, 2] scratch of rows that are
    int64_t rows;
    int cols;
    int split;
};

// Parts that a row of logits is split into where there is scratch for it.
int policy_split(int dtype, int64_t rows, int64_t cols);
void launch_policy_loss(int dtype, const PolicyArgs& a, hipStream_t st);

struct PolicyGradArgs {
    const void* x;
    Dims kept;
    const void* token;
    int token64;
    const float* lse;
    const float* weight;
    float upstream;
    void* out;
    int64_t rows;
    int cols;
};
void launch_policy_loss_backward(int dtype, const PolicyGradArgs& a, hipStream_t st);

}  // namespace hpt
