// C ABI of libhpt_hip (see include/hpt_hip.h): argument validation, the device
// caching allocator, per-stream scratch, and dispatch into the kernel tables.
#include <hip/hip_runtime.h>

#include <atomic>
#include <cmath>
#include <cstring>
#include <memory>
#include <list>
#include <map>
#include <mutex>
#include <optional>
#include <unordered_map>
#include <vector>

#include "block_entry.hpp"
#include "common.hpp"
#include "elementwise_entry.hpp"
#include "norm_entry.hpp"
#include "reduce_entry.hpp"

namespace hpt {

// ---- error transport ---------------------------------------------------------

static thread_local std::string g_last_error;

template <class F> static int32_t guarded(F&& f) {
    try {
        f();
        return HPT_OK;
    } catch (const Error& e) {
        g_last_error = e.msg;
        return e.code;
    } catch (const std::bad_alloc&) {
        g_last_error = "host allocation failed";
        return HPT_ERR_MEMORY;
    } catch (...) {
        g_last_error = "unknown error";
        return HPT_ERR_KERNEL;
    }
}

static void hip_check(hipError_t e, int code, const char* what) {
    if (e != hipSuccess) fail(code, "%s: %s", what, hipGetErrorString(e));
}

// Make `dev` the calling thread's device. The device count is asked for once per process and
// hipSetDevice is skipped when the thread is already there (hipGetDevice reads a thread-local of the
// runtime): on launch-bound calls the two runtime calls this saves are a measurable part of the
// host time.
static void use_device(int dev) {
    static std::atomic<int> count{-1};
    int n = count.load(std::memory_order_relaxed);
    if (n < 0) {
        hip_check(hipGetDeviceCount(&n), HPT_ERR_DEVICE, "hipGetDeviceCount");
        count.store(n, std::memory_order_relaxed);
    }
    if (dev < 0 || dev >= n) fail(HPT_ERR_DEVICE, "device %d does not exist (%d visible)", dev, n);
    int cur = -1;
    if (hipGetDevice(&cur) != hipSuccess || cur != dev)
        hip_check(hipSetDevice(dev), HPT_ERR_DEVICE, "hipSetDevice");
}

// Whether work on `st` is being recorded (or may not be asked about because another stream's is): scratch must
// not be allocated then, and a recorded call outlives the buffer's next owner.
static bool capturing(hipStream_t st) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(st, &status) != hipSuccess) {
        (void)hipGetLastError();
        return true;
    }
    return status != hipStreamCaptureStatusNone;
}

// Lets the calling thread make runtime calls that a capture in progress (its own or another thread's, on streams that
// these calls do not touch) would otherwise refuse.
struct RelaxedCapture {
    hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
    RelaxedCapture() { (void)hipThreadExchangeStreamCaptureMode(&mode); }
    ~RelaxedCapture() { (void)hipThreadExchangeStreamCaptureMode(&mode); }
};

// ---- device caching allocator ------------------------------------------------
// Same policy as the reference's CudaAllocator
// (hpt-allocator/src/allocators/cuda.rs:41-322, utils/allocate.rs:15-130,
// utils/deallocate.rs:11-32): blocks are keyed by their exact (size, align)
// layout; a freed block is kept in an LRU cache of layouts; evicting a layout
// releases all of its blocks; when the device is out of memory, layouts are
// evicted least-recently-used first and the allocation is retried.
// A block may come back while work on the DEFAULT stream still uses it (hpt_hip_free_ordered): it is numbered, and
// handed on at once only to a caller whose first use of it is queued on the same stream (hpt_hip_alloc_ordered), so the
// queue itself keeps the two apart. Anybody else waits for the default stream first, which makes every block numbered
// so far idle. (Waiting at every free instead kept the host and the device taking turns: about 25 us of a pass.)
// That wait lasts as long as the stream has work: it is made without the lock, and ordered callers take blocks in use
// before idle ones, so that whoever needs an idle block mostly finds one.

struct LayoutKey {
    size_t bytes, align;
    bool operator<(const LayoutKey& o) const {
        return bytes != o.bytes ? bytes < o.bytes : align < o.align;
    }
};

struct CachedBlock {
    void* p;
    uint64_t number;  // of the free that left work queued on the default stream; 0: idle
};

struct DeviceAllocator {
    std::mutex mu;
    uint64_t last_number = 0, idle_upto = 0;  // blocks numbered up to idle_upto are known to be idle
    size_t capacity = 100;  // cached layouts; the CPU allocator's default (allocators/cpu.rs:22)
    std::list<LayoutKey> lru;  // front = most recently used
    std::map<LayoutKey, std::pair<std::list<LayoutKey>::iterator, std::vector<CachedBlock>>> cache;
    std::unordered_map<void*, LayoutKey> live;
    uint64_t device_mallocs = 0;
    size_t internal_blocks = 0;  // live blocks the library itself holds (scratch), not a caller

    size_t cached_blocks() const {
        size_t n = 0;
        for (auto& kv : cache) n += kv.second.second.size();
        return n;
    }
    // Requires `mu` and the device to be current. False where the stream cannot be waited for: while another stream
    // that it orders itself with is being captured. `lock` (on mu) is let go for the wait: the cache may be another after.
    bool wait_default_stream(std::unique_lock<std::mutex>* lock = nullptr) {
        const uint64_t upto = last_number;
        if (idle_upto >= upto) return true;
        if (capturing(nullptr)) return false;
        RelaxedCapture relaxed;
        if (lock) lock->unlock();
        const hipError_t e = hipStreamSynchronize(nullptr);
        if (lock) lock->lock();
        if (e != hipSuccess) {
            (void)hipGetLastError();
            return false;
        }
        idle_upto = std::max(idle_upto, upto);
        return true;
    }
    void evict_one() {  // requires a non-empty cache
        LayoutKey k = lru.back();
        auto it = cache.find(k);
        for (const CachedBlock& b : it->second.second) {
            if (b.number > idle_upto) (void)wait_default_stream();
            (void)hipFree(b.p);
        }
        cache.erase(it);
        lru.pop_back();
    }
    // `lock` holds mu. `ordered`: the block's first use will be queued on the default stream.
    void* allocate(std::unique_lock<std::mutex>& lock, size_t bytes, size_t align, bool ordered = false) {
        LayoutKey k{bytes, align};
        auto it = cache.find(k);
        size_t take = 0;  // one more than the index of the block to hand out
        for (bool waited = false; it != cache.end(); waited = true, it = cache.find(k)) {
            const std::vector<CachedBlock>& blocks = it->second.second;
            take = blocks.size();
            while (take && (blocks[take - 1].number > idle_upto) != ordered) --take;
            if (!take && ordered) take = blocks.size();
            if (take || waited || !wait_default_stream(&lock)) break;
        }
        if (take) {
            std::vector<CachedBlock>& blocks = it->second.second;
            void* p = blocks[take - 1].p;
            blocks.erase(blocks.begin() + (take - 1));
            lru.splice(lru.begin(), lru, it->second.first);
            if (it->second.second.empty()) {
                lru.erase(it->second.first);
                cache.erase(it);
            }
            live[p] = k;
            return p;
        }
        void* p = nullptr;
        // Device memory is not allocated while a capture refuses it (scratch least of all: its address would be recorded, and
        // hpt_hip_cache_clear hands it on) - except in the place of a cached block that is only not idle yet.
        std::optional<RelaxedCapture> relaxed;
        if (it != cache.end()) relaxed.emplace();
        for (;;) {
            hipError_t e = hipMalloc(&p, bytes ? bytes : 1);
            if (e == hipSuccess) break;
            (void)hipGetLastError();  // clear the sticky error before retrying
            if (e != hipErrorOutOfMemory || cache.empty())
                fail(HPT_ERR_MEMORY, "Failed to allocate %zu bytes on device: %s", bytes,
                     hipGetErrorString(e));
            evict_one();
        }
        ++device_mallocs;
        if (align > 1 && ((uintptr_t)p % align) != 0) {
            (void)hipFree(p);
            fail(HPT_ERR_MEMORY, "device allocation cannot satisfy alignment %zu", align);
        }
        live[p] = k;
        return p;
    }
    // `ordered`: work queued on the default stream, and on no other, may still use the block.
    void deallocate(void* p, size_t bytes, size_t align, bool ordered = false) {
        auto it = live.find(p);
        if (it == live.end()) fail(HPT_ERR_MEMORY, "pointer %p was not allocated by hpt_hip_alloc", p);
        if (it->second.bytes != bytes || it->second.align != align)
            fail(HPT_ERR_MEMORY, "layout mismatch on free: allocated (%zu, %zu), freed as (%zu, %zu)",
                 it->second.bytes, it->second.align, bytes, align);
        LayoutKey k = it->second;
        live.erase(it);
        const CachedBlock b{p, ordered ? ++last_number : 0};
        if (capacity == 0) {
            if (ordered) (void)wait_default_stream();
            (void)hipFree(p);
            return;
        }
        auto c = cache.find(k);
        if (c == cache.end()) {
            lru.push_front(k);
            cache[k] = {lru.begin(), {b}};
            while (cache.size() > capacity) evict_one();
        } else {
            c->second.second.push_back(b);
            lru.splice(lru.begin(), lru, c->second.first);
        }
    }
    // The caller takes the block over: it leaves the table of live blocks and is not cached.
    bool forget(void* p) { return live.erase(p) != 0; }
    void clear() {
        while (!cache.empty()) evict_one();
    }
};

static std::mutex g_alloc_table_mu;
static std::map<int, DeviceAllocator*> g_allocators;

static DeviceAllocator& allocator_of(int dev) {
    std::lock_guard<std::mutex> g(g_alloc_table_mu);
    auto it = g_allocators.find(dev);
    if (it == g_allocators.end()) it = g_allocators.emplace(dev, new DeviceAllocator()).first;
    return *it->second;
}

// ---- scratch of the multi-workgroup reductions -----------------------------------
// One buffer per (device, stream), taken from the device's caching allocator (so that
// hpt_hip_cache_clear and the evict-and-retry path see it) and guarded by a lock of its own:
// calls on different streams do not wait for each other. It grows geometrically; the buffer it
// outgrows is not handed back while work that uses it may still be queued, but parked until
// hpt_hip_cache_clear, which waits for the device first. No call on the hot path frees device
// memory.

constexpr size_t kScratchAlign = 256;

struct StreamScratch {
    std::mutex mu;  // held from lookup to launch by the call that uses the buffer
    void* base = nullptr;
    size_t bytes = 0;
    std::vector<std::pair<void*, size_t>> retired;
};

static std::mutex g_scratch_table_mu;  // guards the map only
static std::map<std::pair<int, hipStream_t>, std::unique_ptr<StreamScratch>> g_scratch;

static StreamScratch& scratch_entry(int dev, hipStream_t st) {
    std::lock_guard<std::mutex> g(g_scratch_table_mu);
    auto& e = g_scratch[{dev, st}];
    if (!e) e.reset(new StreamScratch());
    return *e;
}

// Requires s.mu. Returns a buffer of at least `bytes`. Nothing in it has to start from a known
// value: every kernel that reads a scratch slot runs after the kernel that wrote it, on this stream.
static void* scratch_reserve(int dev, StreamScratch& s, size_t bytes) {
    if (!s.base || bytes > s.bytes) {
        const size_t want = std::max<size_t>({bytes, s.bytes * 2, (size_t)1 << 20});
        DeviceAllocator& a = allocator_of(dev);
        void* p;
        {
            std::unique_lock<std::mutex> g(a.mu);
            p = a.allocate(g, want, kScratchAlign);
            ++a.internal_blocks;
        }
        if (s.base) s.retired.emplace_back(s.base, s.bytes);
        s.base = p;
        s.bytes = want;
    }
    return s.base;
}

// Give every scratch buffer of `dev` back to its allocator. The table and every buffer of the device are
// locked BEFORE the device is waited for and stay locked until the buffers are back: a call on another thread
// that needs scratch either got its buffer earlier (its kernels are then queued, and waited for here) or
// blocks until this is over and allocates afresh. (Locks are taken table -> buffer -> allocator everywhere.)
static void scratch_release_all(int dev) {
    std::lock_guard<std::mutex> gt(g_scratch_table_mu);
    std::vector<std::unique_lock<std::mutex>> held;
    for (auto& kv : g_scratch)
        if (kv.first.first == dev) held.emplace_back(kv.second->mu);
    hip_check(hipDeviceSynchronize(), HPT_ERR_KERNEL, "hipDeviceSynchronize");
    DeviceAllocator& a = allocator_of(dev);
    for (auto& kv : g_scratch) {
        if (kv.first.first != dev) continue;
        StreamScratch& s = *kv.second;
        std::lock_guard<std::mutex> ga(a.mu);
        if (s.base) s.retired.emplace_back(s.base, s.bytes);
        for (auto& r : s.retired) {
            a.deallocate(r.first, r.second, kScratchAlign);
            --a.internal_blocks;
        }
        s.retired.clear();
        s.base = nullptr;
        s.bytes = 0;
    }
}

size_t scratch_need(const ReducePlan& p, size_t acc_size) {
    return p.split > 1 ? (size_t)p.K * p.split * acc_size : 0;
}

// ---- scratch that is never allocated (hpt_hip_reduce_static) ------------------------
// Part of the library's image on every device it runs on. In host code the array's name
// is only a handle for hipGetSymbolAddress: the device address is looked up once per
// device, with that device current, and only that address is ever handed to a kernel.
constexpr size_t kStaticScratchBytes = HPT_HIP_STATIC_SCRATCH_BYTES;
static __device__ __align__(256) unsigned char scratch[kStaticScratchBytes];

static std::mutex g_static_scratch_mu;
static std::map<int, void*> g_static_scratch_ptr;

// Requires `dev` to be the current device.
static void* static_scratch_of(int dev) {
    std::lock_guard<std::mutex> g(g_static_scratch_mu);
    auto it = g_static_scratch_ptr.find(dev);
    if (it != g_static_scratch_ptr.end()) return it->second;
    void* ptr = nullptr;
    hip_check(hipGetSymbolAddress((void**)&ptr, HIP_SYMBOL(scratch)), HPT_ERR_DEVICE,
              "hipGetSymbolAddress(scratch)");
    if (!ptr) fail(HPT_ERR_DEVICE, "hipGetSymbolAddress(scratch) returned a null address");
    g_static_scratch_ptr.emplace(dev, ptr);
    return ptr;
}

// ---- dispatch tables -----------------------------------------------------------

const ReduceEntry& reduce_entry_for(int e) {
    switch (e) {
        case 0: return reduce_entry<0>();
        case 1: return reduce_entry<1>();
        case 2: return reduce_entry<2>();
        case 3: return reduce_entry<3>();
        case 4: return reduce_entry<4>();
        case 5: return reduce_entry<5>();
        case 6: return reduce_entry<6>();
        case 7: return reduce_entry<7>();
        case 8: return reduce_entry<8>();
        case 9: return reduce_entry<9>();
        case 10: return reduce_entry<10>();
        case 11: return reduce_entry<11>();
        case 12: return reduce_entry<12>();
        case 13: return reduce_entry<13>();
        case 14: return reduce_entry<14>();
        case 15: return reduce_entry<15>();
        default: fail(HPT_ERR_PARAM, "invalid reduce op %d", e);
    }
}

NormLaunchFn norm_launcher_for(int kind, int dtype) {
    switch (kind) {
        case NORM_SOFTMAX: return norm_launcher<NORM_SOFTMAX>(dtype);
        case NORM_LOGSOFTMAX: return norm_launcher<NORM_LOGSOFTMAX>(dtype);
        case NORM_LAYERNORM: return norm_launcher<NORM_LAYERNORM>(dtype);
        case NORM_ADD_LAYERNORM: return norm_launcher<NORM_ADD_LAYERNORM>(dtype);
        case NORM_SOFTMAX_CAUSAL: return norm_launcher<NORM_SOFTMAX_CAUSAL>(dtype);
        case NORM_LOGSOFTMAX_CAUSAL: return norm_launcher<NORM_LOGSOFTMAX_CAUSAL>(dtype);
        default: return nullptr;
    }
}

NormLaunchFn norm_promoting_launcher_for(int kind, int in_dtype) {
    switch (kind) {
        case NORM_SOFTMAX: return norm_promoting_launcher<NORM_SOFTMAX>(in_dtype);
        case NORM_LOGSOFTMAX: return norm_promoting_launcher<NORM_LOGSOFTMAX>(in_dtype);
        case NORM_LAYERNORM: return norm_promoting_launcher<NORM_LAYERNORM>(in_dtype);
        default: return nullptr;  // the fused kinds take float inputs only
    }
}

// ---- view validation -------------------------------------------------------------

static void check_view(const hpt_view* v, const char* name, bool need_data) {
    if (!v) fail(HPT_ERR_PARAM, "%s: view is null", name);
    if (v->dtype < 0 || v->dtype >= HPT_DTYPE_COUNT)
        fail(HPT_ERR_DTYPE, "%s: invalid dtype %d", name, v->dtype);
    if (v->ndim < 0 || v->ndim > kMaxRank)
        fail(HPT_ERR_SHAPE, "%s: ndim %d outside 0..%d", name, v->ndim, kMaxRank);
    if (v->ndim > 0 && (!v->shape || !v->strides))
        fail(HPT_ERR_PARAM, "%s: shape/strides are null", name);
    int64_t n = 1;
    for (int i = 0; i < v->ndim; ++i) {
        if (v->shape[i] < 0) fail(HPT_ERR_SHAPE, "%s: negative dim %lld", name, (long long)v->shape[i]);
        n *= v->shape[i];
    }
    if (need_data && n > 0 && !v->data) fail(HPT_ERR_PARAM, "%s: data pointer is null", name);
}

static int64_t view_size(const hpt_view* v) {
    int64_t n = 1;
    for (int i = 0; i < v->ndim; ++i) n *= v->shape[i];
    return n;
}

// Layout::is_contiguous (hpt-common/src/layout/layout_utils.rs:363-375), with
// size-1 dims allowed any stride.
static bool view_contiguous(const hpt_view* v) {
    int64_t expect = 1;
    for (int i = v->ndim - 1; i >= 0; --i) {
        if (v->shape[i] == 0) return true;
        if (v->shape[i] == 1) continue;
        if (v->strides[i] != expect) return false;
        expect *= v->shape[i];
    }
    return true;
}

static void check_out(const hpt_view* out, int dtype, int64_t count, const char* name) {
    check_view(out, name, true);
    if (out->dtype != dtype)
        fail(HPT_ERR_DTYPE, "%s: dtype is %s, expected %s", name, dtype_name(out->dtype),
             dtype_name(dtype));
    if (!view_contiguous(out)) fail(HPT_ERR_SHAPE, "%s: output tensor must be contiguous", name);
    if (view_size(out) != count)
        fail(HPT_ERR_SHAPE, "%s: Size mismatch: expected %lld, got %lld", name, (long long)count,
             (long long)view_size(out));
}

// The bytes a view can touch: [lo, hi) around its data pointer.
static void view_extent(const hpt_view* v, const char** lo, const char** hi) {
    const int64_t es = (int64_t)dtype_size(v->dtype);
    int64_t below = 0, above = 0;
    for (int i = 0; i < v->ndim; ++i) {
        const int64_t span = (v->shape[i] - 1) * v->strides[i];
        if (span < 0) below += span;
        else above += span;
    }
    *lo = (const char*)v->data + below * es;
    *hi = (const char*)v->data + (above + 1) * es;
}

// `out` must not share memory with `in`. With allow_same, `out` may be `in` itself: the same
// pointer, dtype and contiguous layout, where every element is read before it is written by the
// thread that writes it. Anything else (a permuted, sliced, stepped or shifted view of out's
// buffer) would be read and written in different orders by different workgroups.
static void check_alias(const hpt_view* in, const hpt_view* out, bool allow_same, const char* what,
                        const char* in_name) {
    if (!in || !in->data || !out->data) return;
    if (view_size(in) == 0 || view_size(out) == 0) return;
    const char *ilo, *ihi, *olo, *ohi;
    view_extent(in, &ilo, &ihi);
    view_extent(out, &olo, &ohi);
    if (!(ilo < ohi && olo < ihi)) return;
    bool same = allow_same && in->data == out->data && in->dtype == out->dtype && in->ndim == out->ndim &&
                view_contiguous(in);
    for (int i = 0; same && i < in->ndim; ++i) same = in->shape[i] == out->shape[i];
    if (!same)
        fail(HPT_ERR_PARAM, "%s: out overlaps %s%s", what, in_name,
             allow_same ? " without being that very tensor (same pointer and contiguous layout)" : "");
}

static void check_launch(const char* what) {
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) fail(HPT_ERR_KERNEL, "%s: kernel launch failed: %s", what, hipGetErrorString(e));
}

struct ReduceCall {
    ReducePlan plan;
    const ReduceEntry* entry;
    int out_dtype;
};

static ReduceCall prepare_reduce(int entry_id, const hpt_view* in, const int64_t* axes, int naxes, bool spare_scratch = true) {
    check_view(in, "reduce input", false);
    if (naxes < 0 || naxes > kMaxRank || (naxes > 0 && !axes))
        fail(HPT_ERR_PARAM, "reduce: bad axes argument");
    int64_t norm[kMaxRank];
    process_axes(axes, naxes, in->ndim, norm);
    if (in->ndim == 0) naxes = 0;
    ReduceCall c;
    c.entry = &reduce_entry_for(entry_id);
    c.out_dtype = entry_id < HPT_REDUCE_OP_COUNT ? reduce_out_dtype(entry_id, in->dtype) : HPT_I64;
    // an exponential per element (two-byte results take the hardware exp2: cheap), or squares in f64
    const bool heavy = (entry_id == HPT_LOGSUMEXP && dtype_size(c.out_dtype) > 2) ||
                       ((entry_id == HPT_SUM_SQUARE || entry_id == HPT_REDUCEL2) && in->dtype == HPT_F32);
    c.plan = plan_reduce(in->data, in->shape, in->strides, in->ndim, norm, naxes,
                         dtype_size(in->dtype), c.entry->acc_size[in->dtype], heavy, spare_scratch);
    return c;
}

// use_static: the partials go to the library's static device array instead of allocated
// scratch; a plan that needs more than the array holds is refused.
// Small inputs that are split for speed alone are reduced in one launch where scratch is not to be had for the
// asking: for the static entry (whose one array is shared by all streams), under capture, and when the device is full.
static void run_reduce(int dev, void* stream, int entry_id, const hpt_view* in, const int64_t* axes,
                       int naxes, int init_out, hpt_view* out, bool use_static = false) {
    ReduceCall c = prepare_reduce(entry_id, in, axes, naxes, !use_static);
    check_out(out, c.out_dtype, c.plan.K, "reduce output");
    check_alias(in, out, false, "reduce", "the input");
    if (c.plan.kind == ReduceKind::Empty) return;
    if (!in->data && c.plan.kind != ReduceKind::Identity)
        fail(HPT_ERR_PARAM, "reduce input: data pointer is null");
    if (!init_out && !(entry_id == HPT_SUM || entry_id == HPT_NANSUM))
        fail(HPT_ERR_PARAM, "init_out = 0 (accumulate into out) is only defined for sum and nansum");
    size_t pbytes = scratch_need(c.plan, c.entry->acc_size[in->dtype]);
    if (use_static && pbytes > kStaticScratchBytes)
        fail(HPT_ERR_MEMORY,
             "reduce_static: this reduction needs %zu bytes of scratch, the static scratch holds %zu; "
             "use hpt_hip_reduce",
             pbytes, kStaticScratchBytes);
    use_device(dev);
    hipStream_t st = (hipStream_t)stream;
    ReduceLaunchFn fn = c.entry->launch[in->dtype];
    if (c.plan.small_split && capturing(st)) {
        c = prepare_reduce(entry_id, in, axes, naxes, false);
        pbytes = 0;
    }
    if (pbytes && use_static) {
        ReduceScratch sc;
        sc.partial = static_scratch_of(dev);
        fn(c.plan, in->data, out->data, sc, st, init_out);
        check_launch("reduce_static");
    } else if (pbytes) {
        StreamScratch& s = scratch_entry(dev, st);
        std::lock_guard<std::mutex> g(s.mu);
        ReduceScratch sc;
        try {
            sc.partial = scratch_reserve(dev, s, pbytes);
        } catch (const Error&) {
            if (!c.plan.small_split) throw;
            c = prepare_reduce(entry_id, in, axes, naxes, false);
        }
        fn(c.plan, in->data, out->data, sc, st, init_out);
        check_launch("reduce");
    } else {
        fn(c.plan, in->data, out->data, ReduceScratch{}, st, init_out);
        check_launch("reduce");
    }
}

struct NormCall {
    NormPlan plan;
    NormArgs args;
};

// Output dtype of the normalisations: FloatBinaryType<T> (the input's own dtype for floats).
static int norm_out_dtype(int in_dtype) { return reduce_out_dtype(HPT_MEAN, in_dtype); }

// A non-float input is promoted inside the kernel; the plan is made for the output's element size and
// cut down to what the promoting kernel runs. `float_only`: the fused kinds; `residual`: where the other operand of theirs starts.
static NormCall prepare_norm(const hpt_view* in, const void* out_data, int64_t axis, int n_norm_dims,
                             bool float_only = false, const void* residual = nullptr) {
    check_view(in, "normalize input", false);
    if (float_only && !is_float_dtype(in->dtype))
        fail(HPT_ERR_DTYPE, "this fused normalisation needs a float dtype, got %s", dtype_name(in->dtype));
    if (in->ndim == 0) fail(HPT_ERR_SHAPE, "normalize: input has no dimensions");
    if (n_norm_dims <= 0) {
        int64_t a = axis;
        int64_t na;
        process_axes(&a, 1, in->ndim, &na);
        axis = na;
    } else if (n_norm_dims > in->ndim) {
        fail(HPT_ERR_SHAPE, "layernorm: %d normalized dims but input has %d", n_norm_dims, in->ndim);
    }
    NormCall c;
    c.plan = plan_normalize(in->data, out_data, in->shape, in->strides, in->ndim, axis, n_norm_dims,
                            dtype_size(norm_out_dtype(in->dtype)), float_only, residual);
    if (!is_float_dtype(in->dtype)) restrict_to_row_stream(c.plan);
    NormArgs& a = c.args;
    memset(&a, 0, sizeof a);
    a.in = in->data;
    a.out = const_cast<void*>(out_data);
    a.kept_in = c.plan.kept_in;
    a.kept_out = c.plan.kept_out;
    a.norm_in = c.plan.norm_in;
    a.rows = c.plan.rows;
    a.cols = c.plan.cols;
    a.sa = c.plan.norm_in.n == 1 ? c.plan.norm_in.stride[0] : 0;
    a.out_axis_stride = c.plan.out_axis_stride;
    return c;
}

// Launch a normalisation; plans that need scratch (partial row statistics) get
// the per-stream buffer, held under its lock from lookup to launch. Transposed rows off the vector grid have a form
// without scratch too (one group of lanes per row): it is taken under capture and on a full device.
static void launch_norm(int dev, hipStream_t st, NormLaunchFn fn, NormCall& c, const char* what) {
    const bool spare = c.plan.kind == NormKind::Transposed && c.plan.shift;
    if (spare && capturing(st)) demote_to_generic(c.plan);
    if (c.plan.scratch_bytes) {
        StreamScratch& s = scratch_entry(dev, st);
        std::lock_guard<std::mutex> g(s.mu);
        try {
            c.args.scratch = scratch_reserve(dev, s, c.plan.scratch_bytes);
        } catch (const Error&) {
            if (!spare) throw;
            demote_to_generic(c.plan);
        }
        fn(c.plan, c.args, st);
        check_launch(what);
    } else {
        fn(c.plan, c.args, st);
        check_launch(what);
    }
}

// ---- operators around a transformer's blocks ---------------------------------------

constexpr int64_t kMostCols = (int64_t)1 << 29;  // elements of a row that its kernels index with 32 bits

static void check_block_dtype(const hpt_view* v, const char* name) {
    if (v->dtype != HPT_F16 && v->dtype != HPT_BF16 && v->dtype != HPT_F32)
        fail(HPT_ERR_DTYPE, "%s: dtype is %s, expected f16, bf16 or f32", name, dtype_name(v->dtype));
}

// An operand that is contiguous, of one dtype and one size. `shape_of`: of that shape, too.
static void check_operand(const hpt_view* v, int dtype, int64_t count, const hpt_view* shape_of, const char* name) {
    check_view(v, name, true);
    if (v->dtype != dtype) fail(HPT_ERR_DTYPE, "%s: dtype is %s, expected %s", name, dtype_name(v->dtype), dtype_name(dtype));
    if (!view_contiguous(v)) fail(HPT_ERR_SHAPE, "%s: must be contiguous", name);
    bool same = !shape_of || v->ndim == shape_of->ndim;
    for (int i = 0; same && shape_of && i < v->ndim; ++i) same = v->shape[i] == shape_of->shape[i];
    if (!same) fail(HPT_ERR_SHAPE, "%s: shape differs from the input's", name);
    if (view_size(v) != count)
        fail(HPT_ERR_SHAPE, "%s: Size mismatch: expected %lld, got %lld", name, (long long)count, (long long)view_size(v));
}

// The rows of a view whose last `tail` dims are one run of neighbouring elements: their number and length, and where they start.
struct RowsOf {
    int64_t rows = 1, cols = 1;
    Dims kept;
};
static RowsOf rows_of(const hpt_view* v, int tail, const char* name) {
    RowsOf r;
    const int lead = v->ndim - tail;
    for (int i = 0; i < lead; ++i) r.rows *= v->shape[i];
    for (int i = lead; i < v->ndim; ++i) r.cols *= v->shape[i];
    if (r.rows == 0 || r.cols == 0) return r;
    int64_t expect = 1;
    for (int i = v->ndim - 1; i >= lead; --i) {
        if (v->shape[i] == 1) continue;
        if (v->strides[i] != expect) fail(HPT_ERR_SHAPE, "%s: the elements of a row must be neighbours in memory (contiguous() makes them so)", name);
        expect *= v->shape[i];
    }
    if (r.cols >= kMostCols) fail(HPT_ERR_SHAPE, "%s: rows of %lld elements, fewer than %lld expected", name, (long long)r.cols, (long long)kMostCols);
    Dims& d = r.kept;
    for (int i = 0; i < lead; ++i) {
        if (v->shape[i] == 1) continue;
        if (d.n && d.stride[d.n - 1] == v->strides[i] * v->shape[i]) {
            d.size[d.n - 1] *= v->shape[i];
            d.stride[d.n - 1] = v->strides[i];
            continue;
        }
        if (d.n == kMaxDims) fail(HPT_ERR_SHAPE, "%s: more than %d separate dims of rows", name, kMaxDims);
        d.size[d.n] = v->shape[i];
        d.stride[d.n++] = v->strides[i];
    }
    return r;
}

// What a call writes shares no memory with anything else of the call, but for operands that a result may take the very place of.
struct Overlaps {
    struct Of {
        const hpt_view* v;
        const char* name;
    };
    const char* what;
    Of in[12];
    int n_in = 0;
    void reads(const hpt_view* v, const char* name) {
        if (v) in[n_in++] = {v, name};
    }
    // `may`: operands (two at most) whose place `out` may take
    void writes(const hpt_view* out, const hpt_view* may1 = nullptr, const hpt_view* may2 = nullptr, const hpt_view* may3 = nullptr) {
        if (!out) return;
        for (int i = 0; i < n_in; ++i) check_alias(in[i].v, out, in[i].v == may1 || in[i].v == may2 || in[i].v == may3, what, in[i].name);
        in[n_in++] = {out, "another result"};
    }
};

// Scratch of `bytes` for the launches of `go`: the caller's workspace, or the stream's own buffer, held from lookup to launch. A captured call
// outlives that buffer: it takes the form without scratch (`go(nullptr)`) where there is one, and is refused otherwise.
template <class F> static void with_workspace(int dev, hipStream_t st, const hpt_view* ws, size_t bytes, bool without, const char* what, F&& go) {
    if (!bytes) return go(nullptr);
    if (ws) {
        const size_t have = (size_t)view_size(ws) * dtype_size(ws->dtype);
        if (have < bytes) fail(HPT_ERR_MEMORY, "%s: the workspace holds %zu bytes, %zu are needed", what, have, bytes);
        if ((uintptr_t)ws->data % 16) fail(HPT_ERR_PARAM, "%s: the workspace must be aligned to 16 bytes", what);
        return go(ws->data);
    }
    if (capturing(st)) {
        if (without) return go(nullptr);
        fail(HPT_ERR_MEMORY, "%s: under capture a workspace of %zu bytes must be given", what, bytes);
    }
    StreamScratch& s = scratch_entry(dev, st);
    std::lock_guard<std::mutex> g(s.mu);
    void* p = nullptr;
    try {
        p = scratch_reserve(dev, s, bytes);
    } catch (const Error&) {
        if (!without) throw;
    }
    go(p);
}
static void check_workspace(const hpt_view* ws, const char* name) {
    if (!ws) return;
    check_view(ws, name, true);
    if (!view_contiguous(ws)) fail(HPT_ERR_SHAPE, "%s: must be contiguous", name);
}

static float check_eps(double eps) {
    const float e = (float)eps;
    if (!(e > 0.0f) || e > 3.4e38f) fail(HPT_ERR_PARAM, "rms_norm: eps must be a positive number");
    return e;
}

static void run_rms_norm(int dev, void* stream, const hpt_view* in, const hpt_view* residual, int n_norm_dims, const hpt_view* gamma, double eps,
                         int quant, int64_t group, hpt_view* sum, hpt_view* out, hpt_view* scale) {
    check_view(in, "rms_norm input", true);
    check_block_dtype(in, "rms_norm input");
    if (n_norm_dims <= 0 || n_norm_dims > in->ndim) fail(HPT_ERR_SHAPE, "rms_norm: %d normalized dims but input has %d", n_norm_dims, in->ndim);
    const RowsOf r = rows_of(in, n_norm_dims, "rms_norm input");
    const int64_t count = view_size(in);
    RmsArgs a{};
    a.eps = check_eps(eps);
    if (residual) check_operand(residual, in->dtype, count, in, "rms_norm residual");
    if (gamma) check_operand(gamma, in->dtype, r.cols, nullptr, "rms_norm gamma");
    if (sum && !residual) fail(HPT_ERR_PARAM, "rms_norm: a sum is asked for, but there is no residual");
    if (sum) check_out(sum, in->dtype, count, "rms_norm sum");
    a.group = (int)r.cols;
    if (quant == QUANT_NONE) {
        check_out(out, in->dtype, count, "rms_norm output");
    } else {
        if (quant != QUANT_I8 && quant != QUANT_E4M3) fail(HPT_ERR_PARAM, "rms_norm_quant: invalid format %d", quant);
        check_out(out, quant == QUANT_I8 ? HPT_I8 : HPT_U8, count, "rms_norm_quant output");
        if (group < 0 || group > r.cols || (group > 0 && r.cols % group)) fail(HPT_ERR_SHAPE, "rms_norm_quant: groups of %lld do not divide rows of %lld", (long long)group, (long long)r.cols);
        if (group > 0) a.group = (int)group;
        check_out(scale, HPT_F32, r.cols ? r.rows * (r.cols / a.group) : view_size(scale), "rms_norm_quant scale");
    }
    Overlaps o{quant == QUANT_NONE ? "rms_norm" : "rms_norm_quant"};
    o.reads(in, "the input");
    o.reads(residual, "the residual");
    o.reads(gamma, "gamma");
    o.writes(sum, in, residual);
    o.writes(out, in, residual);
    o.writes(scale);
    if (count == 0) return;
    a.x = in->data;
    a.kept = r.kept;
    a.res = residual ? residual->data : nullptr;
    a.gamma = gamma ? gamma->data : nullptr;
    a.sum = sum ? sum->data : nullptr;
    a.out = out->data;
    a.scale = scale ? (float*)scale->data : nullptr;
    a.rows = r.rows;
    a.cols = (int)r.cols;
    use_device(dev);
    launch_rms_norm(in->dtype, quant, a, (hipStream_t)stream);
    check_launch("rms_norm");
}

static RowsOf check_rms_backward(const hpt_view* in, int n_norm_dims) {
    check_view(in, "rms_norm_backward input", true);
    check_block_dtype(in, "rms_norm_backward input");
    if (n_norm_dims <= 0 || n_norm_dims > in->ndim) fail(HPT_ERR_SHAPE, "rms_norm_backward: %d normalized dims but input has %d", n_norm_dims, in->ndim);
    const RowsOf r = rows_of(in, n_norm_dims, "rms_norm_backward input");
    // (no rows are of any length, but gamma has a gradient of zeros)
    if (r.cols >= kMostCols) fail(HPT_ERR_SHAPE, "rms_norm_backward input: rows of %lld elements, fewer than %lld expected", (long long)r.cols, (long long)kMostCols);
    return r;
}
static size_t rms_backward_bytes(const hpt_view* in, const RowsOf& r) {
    return r.rows && r.cols ? (size_t)(rms_grad_partials(in->dtype, r.rows, r.cols) * r.cols) * sizeof(float) : 0;
}

// The scores or probabilities of attention: [..., heads, queries, keys].
struct Scores {
    int64_t batch = 1, heads, queries, keys, rows;
};
static Scores scores_of(const hpt_view* v, const char* name) {
    check_view(v, name, true);
    check_block_dtype(v, name);
    if (v->ndim < 3) fail(HPT_ERR_SHAPE, "%s: needs at least 3 dims (heads x queries x keys)", name);
    Scores s;
    for (int i = 0; i + 3 < v->ndim; ++i) s.batch *= v->shape[i];
    s.heads = v->shape[v->ndim - 3];
    s.queries = v->shape[v->ndim - 2];
    s.keys = v->shape[v->ndim - 1];
    s.rows = s.batch * s.heads * s.queries;
    return s;
}
static float check_bias_scale(double scale, int64_t query_offset, const char* what) {
    if (!(std::abs((float)scale) <= 3.4028234e38f)) fail(HPT_ERR_PARAM, "%s: scale must be a finite number", what);
    if (query_offset < -((int64_t)1 << 40) || query_offset > ((int64_t)1 << 40)) fail(HPT_ERR_PARAM, "%s: query_offset %lld beyond 2^40", what, (long long)query_offset);
    return (float)scale;
}
static void check_lengths(const hpt_view* lengths, const Scores& s, const char* name) {
    if (!lengths) return;
    check_view(lengths, name, true);
    if (lengths->dtype != HPT_I32 && lengths->dtype != HPT_I64) fail(HPT_ERR_DTYPE, "%s: dtype is %s, expected i32 or i64", name, dtype_name(lengths->dtype));
    check_operand(lengths, lengths->dtype, s.batch, nullptr, name);
}

// Logits [..., vocabulary] and a token for each row.
static RowsOf logits_of(const hpt_view* logits, const char* name) {
    check_view(logits, name, true);
    check_block_dtype(logits, name);
    if (logits->ndim < 1) fail(HPT_ERR_SHAPE, "%s: input has no dimensions", name);
    const RowsOf r = rows_of(logits, 1, name);
    if (r.cols == 0) fail(HPT_ERR_SHAPE, "%s: a vocabulary of no tokens", name);
    return r;
}
static void check_tokens(const hpt_view* token, int64_t rows, const char* name) {
    check_view(token, name, true);
    if (token->dtype != HPT_I32 && token->dtype != HPT_I64) fail(HPT_ERR_DTYPE, "%s: dtype is %s, expected i32 or i64", name, dtype_name(token->dtype));
    check_operand(token, token->dtype, rows, nullptr, name);
}
// The parts of split rows, or each token's loss and slope (policy loss only).
static size_t policy_bytes(const hpt_view* logits, const RowsOf& r, bool losses) {
    const int split = policy_split(logits->dtype, r.rows, r.cols);
    return sizeof(double) * (size_t)(split > 1 ? 2 * r.rows * split : losses ? 2 * r.rows : 0);
}
static void run_policy(int dev, void* stream, const hpt_view* logits, const RowsOf& r, PolicyArgs& a, const hpt_view* token, const hpt_view* workspace, bool losses, const char* what) {
    a.x = logits->data;
    a.kept = r.kept;
    a.token = token->data;
    a.token64 = token->dtype == HPT_I64;
    a.rows = r.rows;
    a.cols = (int)r.cols;
    use_device(dev);
    hipStream_t st = (hipStream_t)stream;
    with_workspace(dev, st, workspace, policy_bytes(logits, r, losses), !losses, what, [&](void* p) {
        a.split = p ? policy_split(logits->dtype, r.rows, r.cols) : 1;
        a.each = a.partial = (double*)p;
        launch_policy_loss(logits->dtype, a, st);
        check_launch(what);
    });
}

}  // namespace hpt

using namespace hpt;

extern "C" {

const char* hpt_hip_last_error(void) { return g_last_error.c_str(); }

size_t hpt_hip_dtype_size(int32_t dtype) { return dtype_size(dtype); }

int32_t hpt_hip_device_count(int32_t* n) {
    return guarded([&] {
        if (!n) fail(HPT_ERR_PARAM, "device_count: null output");
        int c = 0;
        hip_check(hipGetDeviceCount(&c), HPT_ERR_DEVICE, "hipGetDeviceCount");
        *n = c;
    });
}

int32_t hpt_hip_alloc(int32_t dev, size_t bytes, size_t align, int32_t zeroed, void** out) {
    return guarded([&] {
        if (!out) fail(HPT_ERR_PARAM, "alloc: null output");
        if (align == 0 || (align & (align - 1))) fail(HPT_ERR_PARAM, "alloc: align %zu is not a power of two", align);
        use_device(dev);
        DeviceAllocator& a = allocator_of(dev);
        std::unique_lock<std::mutex> g(a.mu);
        void* p = a.allocate(g, bytes, align);
        if (zeroed && bytes) {
            hipError_t e = hipMemset(p, 0, bytes);
            if (e != hipSuccess) {
                a.deallocate(p, bytes, align);
                hip_check(e, HPT_ERR_MEMORY, "hipMemset");
            }
        }
        *out = p;
    });
}

int32_t hpt_hip_free(int32_t dev, void* p, size_t bytes, size_t align) {
    return guarded([&] {
        if (!p) return;
        use_device(dev);
        DeviceAllocator& a = allocator_of(dev);
        std::lock_guard<std::mutex> g(a.mu);
        a.deallocate(p, bytes, align);
    });
}

int32_t hpt_hip_alloc_ordered(int32_t dev, size_t bytes, size_t align, void** out) {
    return guarded([&] {
        if (!out) fail(HPT_ERR_PARAM, "alloc: null output");
        if (align == 0 || (align & (align - 1))) fail(HPT_ERR_PARAM, "alloc: align %zu is not a power of two", align);
        use_device(dev);
        DeviceAllocator& a = allocator_of(dev);
        std::unique_lock<std::mutex> g(a.mu);
        *out = a.allocate(g, bytes, align, true);
    });
}

int32_t hpt_hip_free_ordered(int32_t dev, void* p, size_t bytes, size_t align) {
    return guarded([&] {
        if (!p) return;
        use_device(dev);
        DeviceAllocator& a = allocator_of(dev);
        std::lock_guard<std::mutex> g(a.mu);
        a.deallocate(p, bytes, align, true);
    });
}

int32_t hpt_hip_forget(int32_t dev, void* p) {
    return guarded([&] {
        if (!p) return;
        use_device(dev);  // (validates `dev`, as hpt_hip_free does)
        DeviceAllocator& a = allocator_of(dev);
        std::lock_guard<std::mutex> g(a.mu);
        (void)a.forget(p);  // a pointer the allocator does not know is left alone, as in the reference
    });
}

int32_t hpt_hip_cache_resize(int32_t dev, size_t entries) {
    return guarded([&] {
        use_device(dev);
        DeviceAllocator& a = allocator_of(dev);
        std::lock_guard<std::mutex> g(a.mu);
        a.capacity = entries;
        while (a.cache.size() > a.capacity) a.evict_one();
    });
}

int32_t hpt_hip_cache_clear(int32_t dev) {
    return guarded([&] {
        use_device(dev);
        // the scratch buffers go back first (work that uses them may still be queued: waited for inside)
        scratch_release_all(dev);
        DeviceAllocator& a = allocator_of(dev);
        std::lock_guard<std::mutex> g(a.mu);
        a.clear();
    });
}

int32_t hpt_hip_alloc_stats(int32_t dev, uint64_t* live_blocks, uint64_t* cached_blocks,
                            uint64_t* device_mallocs) {
    return guarded([&] {
        DeviceAllocator& a = allocator_of(dev);
        std::lock_guard<std::mutex> g(a.mu);
        if (live_blocks) *live_blocks = a.live.size() - a.internal_blocks;
        if (cached_blocks) *cached_blocks = a.cached_blocks();
        if (device_mallocs) *device_mallocs = a.device_mallocs;
    });
}

int32_t hpt_hip_memcpy_h2d_sync(int32_t dev, void* dst, const void* src, size_t bytes) {
    return guarded([&] {
        if (!bytes) return;
        if (!dst || !src) fail(HPT_ERR_PARAM, "memcpy: null pointer");
        use_device(dev);
        hip_check(hipMemcpy(dst, src, bytes, hipMemcpyHostToDevice), HPT_ERR_DEVICE, "hipMemcpy(h2d)");
    });
}

int32_t hpt_hip_memcpy_d2h_sync(int32_t dev, void* dst, const void* src, size_t bytes) {
    return guarded([&] {
        if (!bytes) return;
        if (!dst || !src) fail(HPT_ERR_PARAM, "memcpy: null pointer");
        use_device(dev);
        hip_check(hipMemcpy(dst, src, bytes, hipMemcpyDeviceToHost), HPT_ERR_DEVICE, "hipMemcpy(d2h)");
    });
}

int32_t hpt_hip_memcpy_d2d_sync(int32_t dev, void* dst, const void* src, size_t bytes) {
    return guarded([&] {
        if (!bytes) return;
        if (!dst || !src) fail(HPT_ERR_PARAM, "memcpy: null pointer");
        use_device(dev);
        hip_check(hipMemcpy(dst, src, bytes, hipMemcpyDeviceToDevice), HPT_ERR_DEVICE, "hipMemcpy(d2d)");
    });
}

int32_t hpt_hip_stream_synchronize(int32_t dev, void* stream) {
    return guarded([&] {
        use_device(dev);
        hip_check(hipStreamSynchronize((hipStream_t)stream), HPT_ERR_KERNEL, "hipStreamSynchronize");
    });
}

int32_t hpt_hip_device_synchronize(int32_t dev) {
    return guarded([&] {
        use_device(dev);
        hip_check(hipDeviceSynchronize(), HPT_ERR_KERNEL, "hipDeviceSynchronize");
    });
}

int32_t hpt_hip_process_axes(const int64_t* axes, int32_t naxes, int32_t ndim, int64_t* out) {
    return guarded([&] {
        if (naxes < 0 || (naxes > 0 && (!axes || !out))) fail(HPT_ERR_PARAM, "process_axes: bad arguments");
        process_axes(axes, naxes, ndim, out);
    });
}

int32_t hpt_hip_reduce_shape(const int64_t* shape, int32_t ndim, const int64_t* axes, int32_t naxes,
                             int32_t keep_dims, int64_t* out_shape, int32_t* out_ndim) {
    return guarded([&] {
        if (ndim < 0 || ndim > kMaxRank || naxes < 0 || naxes > kMaxRank || !out_shape || !out_ndim)
            fail(HPT_ERR_PARAM, "reduce_shape: bad arguments");
        int64_t norm[kMaxRank];
        process_axes(axes, naxes, ndim, norm);
        bool red[kMaxRank] = {};
        if (ndim > 0)
            for (int i = 0; i < naxes; ++i) red[norm[i]] = true;
        int n = 0;
        for (int i = 0; i < ndim; ++i) {
            if (red[i]) {
                if (keep_dims) out_shape[n++] = 1;
            } else {
                out_shape[n++] = shape[i];
            }
        }
        if (n == 0) out_shape[n++] = 1;
        *out_ndim = n;
    });
}

int32_t hpt_hip_reduce_out_dtype(int32_t op, int32_t in_dtype, int32_t* out_dtype) {
    return guarded([&] {
        if (!out_dtype) fail(HPT_ERR_PARAM, "reduce_out_dtype: null output");
        if (op < 0 || op >= HPT_REDUCE_OP_COUNT) fail(HPT_ERR_PARAM, "invalid reduce op %d", op);
        *out_dtype = reduce_out_dtype(op, in_dtype);
    });
}

int32_t hpt_hip_reduce_plan(int32_t op, const hpt_view* in, const int64_t* axes, int32_t naxes,
                            char* buf, size_t buflen) {
    return guarded([&] {
        if (!buf || !buflen) fail(HPT_ERR_PARAM, "reduce_plan: no buffer");
        if (op < 0 || op >= kReduceEntryCount) fail(HPT_ERR_PARAM, "invalid reduce op %d", op);
        ReduceCall c = prepare_reduce(op, in, axes, naxes);
        snprintf(buf, buflen, "%s", describe(c.plan).c_str());
    });
}

int32_t hpt_hip_normalize_plan(const hpt_view* in, int64_t axis, int32_t n_norm_dims, char* buf,
                               size_t buflen) {
    return guarded([&] {
        if (!buf || !buflen) fail(HPT_ERR_PARAM, "normalize_plan: no buffer");
        NormCall c = prepare_norm(in, nullptr, axis, n_norm_dims);
        snprintf(buf, buflen, "%s", describe(c.plan).c_str());
    });
}

int32_t hpt_hip_reduce(int32_t dev, void* stream, int32_t op, const hpt_view* in, const int64_t* axes,
                       int32_t naxes, int32_t init_out, hpt_view* out) {
    return guarded([&] {
        if (op < 0 || op >= HPT_REDUCE_OP_COUNT) fail(HPT_ERR_PARAM, "invalid reduce op %d", op);
        run_reduce(dev, stream, op, in, axes, naxes, init_out, out);
    });
}

int32_t hpt_hip_reduce_static(int32_t dev, void* stream, int32_t op, const hpt_view* in, const int64_t* axes,
                              int32_t naxes, int32_t init_out, hpt_view* out) {
    return guarded([&] {
        if (op < 0 || op >= HPT_REDUCE_OP_COUNT) fail(HPT_ERR_PARAM, "invalid reduce op %d", op);
        run_reduce(dev, stream, op, in, axes, naxes, init_out, out, true);
    });
}

int32_t hpt_hip_argreduce(int32_t dev, void* stream, int32_t is_max, const hpt_view* in, int64_t axis,
                          hpt_view* out) {
    return guarded([&] {
        check_view(in, "argreduce input", false);
        if (in->ndim == 0) fail(HPT_ERR_SHAPE, "argreduce: input has no dimensions");
        int64_t na;
        process_axes(&axis, 1, in->ndim, &na);
        if (in->shape[na] > INT32_MAX)
            fail(HPT_ERR_SHAPE, "argreduce: axis of %lld elements exceeds 2^31-1", (long long)in->shape[na]);
        run_reduce(dev, stream, is_max ? kArgMaxEntry : kArgMinEntry, in, &na, 1, 1, out);
    });
}

int32_t hpt_hip_softmax(int32_t dev, void* stream, int32_t log, const hpt_view* in, int64_t axis,
                        hpt_view* out) {
    return guarded([&] {
        check_view(in, "softmax input", true);
        check_out(out, norm_out_dtype(in->dtype), view_size(in), "softmax output");
        check_alias(in, out, true, "softmax", "the input");
        NormCall c = prepare_norm(in, out->data, axis, 0);
        if (c.plan.kind == NormKind::Empty) return;
        const int kind = log ? NORM_LOGSOFTMAX : NORM_SOFTMAX;
        NormLaunchFn fn = is_float_dtype(in->dtype) ? norm_launcher_for(kind, in->dtype)
                                                    : norm_promoting_launcher_for(kind, in->dtype);
        if (!fn) fail(HPT_ERR_DTYPE, "softmax: unsupported dtype %s", dtype_name(in->dtype));
        use_device(dev);
        launch_norm(dev, (hipStream_t)stream, fn, c, "softmax");
    });
}

// layernorm, optionally of (in + residual)
static void run_layernorm(int dev, void* stream, const hpt_view* in, const hpt_view* residual, int n_norm_dims,
                          const hpt_view* gamma, const hpt_view* beta, double eps, hpt_view* out) {
    check_view(in, "layernorm input", true);
    if (n_norm_dims <= 0) fail(HPT_ERR_SHAPE, "layernorm: normalized_shape must not be empty");
    const int odt = norm_out_dtype(in->dtype);
    check_out(out, odt, view_size(in), "layernorm output");
    check_alias(in, out, true, "layernorm", "the input");
    NormCall c = prepare_norm(in, out->data, 0, n_norm_dims, residual != nullptr, residual ? residual->data : nullptr);
    const hpt_view* gb[2] = {gamma, beta};
    const char* names[2] = {"layernorm gamma", "layernorm beta"};
    for (int k = 0; k < 2; ++k) {
        if (!gb[k]) continue;
        check_view(gb[k], names[k], true);
        if (gb[k]->dtype != odt)
            fail(HPT_ERR_DTYPE, "%s: dtype is %s, expected %s", names[k], dtype_name(gb[k]->dtype),
                 dtype_name(odt));
        if (!view_contiguous(gb[k])) fail(HPT_ERR_SHAPE, "%s: must be contiguous", names[k]);
        check_alias(gb[k], out, false, "layernorm", k == 0 ? "gamma" : "beta");
        // shape must equal the normalised dims (leading 1s aside)
        if (view_size(gb[k]) != c.plan.cols && c.plan.kind != NormKind::Empty)
            fail(HPT_ERR_SHAPE, "%s: Size mismatch: expected %lld, got %lld", names[k],
                 (long long)c.plan.cols, (long long)view_size(gb[k]));
    }
    if (residual) {
        check_view(residual, "layernorm residual", true);
        if (residual->dtype != in->dtype)
            fail(HPT_ERR_DTYPE, "layernorm residual: dtype is %s, expected %s", dtype_name(residual->dtype),
                 dtype_name(in->dtype));
        if (!view_contiguous(residual)) fail(HPT_ERR_SHAPE, "layernorm residual: must be contiguous");
        bool same = residual->ndim == in->ndim;
        for (int i = 0; same && i < in->ndim; ++i) same = residual->shape[i] == in->shape[i];
        if (!same) fail(HPT_ERR_SHAPE, "layernorm residual: shape differs from the input's");
        check_alias(residual, out, true, "layernorm", "the residual");
    }
    if (c.plan.kind == NormKind::Empty) return;
    c.args.gamma = gamma ? gamma->data : nullptr;
    c.args.beta = beta ? beta->data : nullptr;
    c.args.residual = residual ? residual->data : nullptr;
    c.args.eps = eps;
    // the fused form runs on the row kernels only
    if (residual && (c.plan.kind == NormKind::Transposed || c.plan.kind == NormKind::TransposedTile))
        demote_to_generic(c.plan);
    // shifted rows: the residual's rows must be misaligned like the output's
    if (c.plan.shift && !c.plan.ua_rows && residual && (((uintptr_t)residual->data ^ (uintptr_t)out->data) & 15) != 0) demote_to_generic(c.plan);
    // vector loads of gamma / beta / residual need 16-byte alignment too (the shifted streaming
    // kernel reads gamma / beta element by element and the residual with the rows' own shift)
    if (c.plan.vec > 1 && !c.plan.shift &&
        (((uintptr_t)c.args.gamma | (uintptr_t)c.args.beta | (uintptr_t)c.args.residual) % 16) != 0)
        demote_to_generic(c.plan);
    NormLaunchFn fn = is_float_dtype(in->dtype)
                          ? norm_launcher_for(residual ? NORM_ADD_LAYERNORM : NORM_LAYERNORM, in->dtype)
                          : norm_promoting_launcher_for(NORM_LAYERNORM, in->dtype);
    if (!fn) fail(HPT_ERR_DTYPE, "layernorm: unsupported dtype %s", dtype_name(in->dtype));
    use_device(dev);
    launch_norm(dev, (hipStream_t)stream, fn, c, "layernorm");
}

int32_t hpt_hip_layernorm(int32_t dev, void* stream, const hpt_view* in, int32_t n_norm_dims,
                          const hpt_view* gamma, const hpt_view* beta, double eps, hpt_view* out) {
    return guarded([&] { run_layernorm(dev, stream, in, nullptr, n_norm_dims, gamma, beta, eps, out); });
}

int32_t hpt_hip_add_layernorm(int32_t dev, void* stream, const hpt_view* in, const hpt_view* residual,
                              int32_t n_norm_dims, const hpt_view* gamma, const hpt_view* beta, double eps,
                              hpt_view* out) {
    return guarded([&] {
        if (!residual) fail(HPT_ERR_PARAM, "add_layernorm: residual is null");
        run_layernorm(dev, stream, in, residual, n_norm_dims, gamma, beta, eps, out);
    });
}

int32_t hpt_hip_softmax_causal(int32_t dev, void* stream, int32_t log, const hpt_view* in, double scale,
                               int64_t causal_offset, hpt_view* out) {
    return guarded([&] {
        check_view(in, "softmax_causal input", true);
        check_out(out, in->dtype, view_size(in), "softmax_causal output");
        check_alias(in, out, true, "softmax_causal", "the input");
        if (in->ndim < 2) fail(HPT_ERR_SHAPE, "softmax_causal: needs at least 2 dims (queries x keys)");
        NormCall c = prepare_norm(in, out->data, in->ndim - 1, 0, true);
        if (c.plan.kind == NormKind::Empty) return;
        if (c.plan.kind == NormKind::Transposed || c.plan.kind == NormKind::TransposedTile ||
            c.plan.kind == NormKind::ColSplit || c.plan.kind == NormKind::RowSplit || c.plan.kind == NormKind::ColReg)
            demote_to_generic(c.plan);
        c.args.scale = scale;
        c.args.q_rows = in->shape[in->ndim - 2];
        c.args.causal_offset = causal_offset;
        NormLaunchFn fn = norm_launcher_for(log ? NORM_LOGSOFTMAX_CAUSAL : NORM_SOFTMAX_CAUSAL, in->dtype);
        if (!fn) fail(HPT_ERR_DTYPE, "softmax_causal: unsupported dtype %s", dtype_name(in->dtype));
        use_device(dev);
        launch_norm(dev, (hipStream_t)stream, fn, c, "softmax_causal");
    });
}

// ---- the steps either side of the path ------------------------------------------------

static void check_same_shape(const hpt_view* a, const hpt_view* b, const char* what) {
    bool same = a->ndim == b->ndim;
    for (int i = 0; same && i < a->ndim; ++i) same = a->shape[i] == b->shape[i];
    if (!same) fail(HPT_ERR_SHAPE, "%s: shapes differ", what);
}

static EwPlan prepare_copy(const hpt_view* in, const hpt_view* out) {
    check_view(in, "contiguous input", true);
    check_out(out, in->dtype, view_size(in), "contiguous output");
    check_same_shape(in, out, "contiguous");
    check_alias(in, out, false, "contiguous", "the input");
    const void* datas[1] = {in->data};
    const int64_t* strides[1] = {in->strides};
    return plan_elementwise(out->data, in->shape, in->ndim, 1, datas, strides, dtype_size(in->dtype), true);
}

int32_t hpt_hip_contiguous(int32_t dev, void* stream, const hpt_view* in, hpt_view* out) {
    return guarded([&] {
        const EwPlan p = prepare_copy(in, out);
        if (p.kind == EwKind::Empty) return;
        use_device(dev);
        launch_strided_copy(in->dtype, p, out->data, in->data, (hipStream_t)stream);
        check_launch("contiguous");
    });
}

int32_t hpt_hip_contiguous_plan(const hpt_view* in, const hpt_view* out, char* buf, size_t buflen) {
    return guarded([&] {
        if (!buf || !buflen) fail(HPT_ERR_PARAM, "contiguous_plan: no buffer");
        snprintf(buf, buflen, "%s", describe(prepare_copy(in, out)).c_str());
    });
}

int32_t hpt_hip_cast(int32_t dev, void* stream, const hpt_view* in, hpt_view* out) {
    return guarded([&] {
        check_view(in, "cast input", true);
        check_view(out, "cast output", true);
        if (!view_contiguous(out)) fail(HPT_ERR_SHAPE, "cast output: output tensor must be contiguous");
        check_same_shape(in, out, "cast");
        check_alias(in, out, false, "cast", "the input");
        if (in->dtype == out->dtype) {
            const EwPlan p = prepare_copy(in, out);
            if (p.kind == EwKind::Empty) return;
            use_device(dev);
            launch_strided_copy(in->dtype, p, out->data, in->data, (hipStream_t)stream);
            check_launch("cast");
            return;
        }
        const size_t es = std::max(dtype_size(in->dtype), dtype_size(out->dtype));
        const void* datas[1] = {in->data};
        const int64_t* strides[1] = {in->strides};
        const EwPlan p = plan_elementwise(out->data, in->shape, in->ndim, 1, datas, strides, es, false);
        if (p.kind == EwKind::Empty) return;
        use_device(dev);
        launch_cast(in->dtype, out->dtype, p, out->data, in->data, (hipStream_t)stream);
        check_launch("cast");
    });
}

int32_t hpt_hip_fill(int32_t dev, void* stream, hpt_view* out, const void* value) {
    return guarded([&] {
        check_view(out, "fill output", true);
        if (!view_contiguous(out)) fail(HPT_ERR_SHAPE, "fill output: output tensor must be contiguous");
        if (!value) fail(HPT_ERR_PARAM, "fill: value pointer is null");
        const int64_t n = view_size(out);
        if (n == 0) return;
        use_device(dev);
        launch_fill(out->dtype, out->data, n, value, (hipStream_t)stream);
        check_launch("fill");
    });
}

// Argument checks of a binary op and the plan its kernels run.
static EwPlan prepare_binary(const hpt_view* lhs, const hpt_view* rhs, const hpt_view* out) {
    check_view(lhs, "binary lhs", true);
    check_view(rhs, "binary rhs", true);
    if (lhs->dtype != rhs->dtype)
        fail(HPT_ERR_DTYPE, "binary: operands must share one dtype, got %s and %s", dtype_name(lhs->dtype),
             dtype_name(rhs->dtype));
    check_out(out, lhs->dtype, view_size(lhs), "binary output");
    check_same_shape(lhs, out, "binary lhs / out");
    check_same_shape(rhs, out, "binary rhs / out");
    // The output may be one of the operands (in place) but must not overlap one otherwise:
    // every element is read before it is written only when the two walk the same addresses.
    check_alias(lhs, out, true, "binary", "lhs");
    check_alias(rhs, out, true, "binary", "rhs");
    const void* datas[2] = {lhs->data, rhs->data};
    const int64_t* strides[2] = {lhs->strides, rhs->strides};
    return plan_elementwise(out->data, out->shape, out->ndim, 2, datas, strides, dtype_size(out->dtype), true);
}

int32_t hpt_hip_binary(int32_t dev, void* stream, int32_t op, const hpt_view* lhs, const hpt_view* rhs,
                       hpt_view* out) {
    return guarded([&] {
        const EwPlan p = prepare_binary(lhs, rhs, out);
        if (p.kind == EwKind::Empty) return;
        use_device(dev);
        launch_binary(op, out->dtype, p, out->data, lhs->data, rhs->data, (hipStream_t)stream);
        check_launch("binary");
    });
}

int32_t hpt_hip_binary_plan(const hpt_view* lhs, const hpt_view* rhs, const hpt_view* out, char* buf, size_t buflen) {
    return guarded([&] {
        if (!buf || !buflen) fail(HPT_ERR_PARAM, "binary_plan: no buffer");
        snprintf(buf, buflen, "%s", describe(prepare_binary(lhs, rhs, out)).c_str());
    });
}

// ---- operators around a transformer's blocks ------------------------------------------

int32_t hpt_hip_rms_norm(int32_t dev, void* stream, const hpt_view* in, const hpt_view* residual, int32_t n_norm_dims,
                         const hpt_view* gamma, double eps, hpt_view* sum, hpt_view* out) {
    return guarded([&] { run_rms_norm(dev, stream, in, residual, n_norm_dims, gamma, eps, QUANT_NONE, 0, sum, out, nullptr); });
}

int32_t hpt_hip_rms_norm_quant(int32_t dev, void* stream, const hpt_view* in, const hpt_view* residual, int32_t n_norm_dims,
                               const hpt_view* gamma, double eps, int32_t format, int64_t group, hpt_view* sum, hpt_view* out,
                               hpt_view* scale) {
    return guarded([&] {
        if (format != HPT_QUANT_I8 && format != HPT_QUANT_E4M3) fail(HPT_ERR_PARAM, "rms_norm_quant: invalid format %d", format);
        if (!scale) fail(HPT_ERR_PARAM, "rms_norm_quant scale: view is null");
        run_rms_norm(dev, stream, in, residual, n_norm_dims, gamma, eps, format == HPT_QUANT_I8 ? QUANT_I8 : QUANT_E4M3, group, sum, out, scale);
    });
}

int32_t hpt_hip_rms_norm_backward_workspace(const hpt_view* in, int32_t n_norm_dims, size_t* bytes) {
    return guarded([&] {
        if (!bytes) fail(HPT_ERR_PARAM, "rms_norm_backward_workspace: null output");
        *bytes = rms_backward_bytes(in, check_rms_backward(in, n_norm_dims));
    });
}

int32_t hpt_hip_rms_norm_backward(int32_t dev, void* stream, const hpt_view* in, const hpt_view* grad, const hpt_view* grad_sum,
                                  int32_t n_norm_dims, const hpt_view* gamma, double eps, const hpt_view* workspace, hpt_view* grad_in,
                                  hpt_view* grad_gamma) {
    return guarded([&] {
        const RowsOf r = check_rms_backward(in, n_norm_dims);
        const int64_t count = view_size(in);
        RmsGradArgs a{};
        a.eps = check_eps(eps);
        check_operand(grad, in->dtype, count, in, "rms_norm_backward grad");
        if (grad_sum) check_operand(grad_sum, in->dtype, count, in, "rms_norm_backward grad_sum");
        if (gamma) check_operand(gamma, in->dtype, r.cols, nullptr, "rms_norm_backward gamma");
        check_workspace(workspace, "rms_norm_backward workspace");
        check_out(grad_in, in->dtype, count, "rms_norm_backward grad_in");
        if (grad_gamma) check_out(grad_gamma, HPT_F32, r.cols, "rms_norm_backward grad_gamma");
        Overlaps o{"rms_norm_backward"};
        o.reads(in, "the input");
        o.reads(grad, "grad");
        o.reads(grad_sum, "grad_sum");
        o.reads(gamma, "gamma");
        o.writes(grad_in, in, grad, grad_sum);
        o.writes(grad_gamma);
        if (workspace) {
            hpt_view w = *workspace;
            o.writes(&w);
        }
        if (r.cols == 0 || (count == 0 && !grad_gamma)) return;
        a.x = in->data;
        a.kept = r.kept;
        a.gy = grad->data;
        a.gsum = grad_sum ? grad_sum->data : nullptr;
        a.gamma = gamma ? gamma->data : nullptr;
        a.gx = grad_in->data;
        a.ggamma = grad_gamma ? (float*)grad_gamma->data : nullptr;
        a.rows = r.rows;
        a.cols = (int)r.cols;
        use_device(dev);
        hipStream_t st = (hipStream_t)stream;
        with_workspace(dev, st, workspace, grad_gamma ? rms_backward_bytes(in, r) : 0, false, "rms_norm_backward", [&](void* p) {
            a.partial = (float*)p;
            launch_rms_norm_backward(in->dtype, a, st);
            check_launch("rms_norm_backward");
        });
    });
}

int32_t hpt_hip_softmax_bias_workspace(const hpt_view* in, size_t* bytes) {
    return guarded([&] {
        if (!bytes) fail(HPT_ERR_PARAM, "softmax_bias_workspace: null output");
        const Scores s = scores_of(in, "softmax_bias input");
        const int split = bias_split(in->dtype, s.rows, s.keys);
        *bytes = split > 1 ? (size_t)(s.rows * split) * 2 * sizeof(float) : 0;
    });
}

int32_t hpt_hip_softmax_bias(int32_t dev, void* stream, const hpt_view* in, double scale, const hpt_view* table, int32_t bidirectional,
                             int64_t max_distance, int64_t query_offset, int32_t causal, const hpt_view* lengths,
                             const hpt_view* workspace, hpt_view* out) {
    return guarded([&] {
        const Scores s = scores_of(in, "softmax_bias input");
        (void)rows_of(in, 1, "softmax_bias input");  // (keys side by side, fewer than 2^29)
        hpt_view heads = *in;
        heads.ndim = in->ndim - 2;
        const RowsOf r = rows_of(&heads, 0, "softmax_bias input");
        BiasArgs a{};
        a.scale = check_bias_scale(scale, query_offset, "softmax_bias");
        check_view(table, "softmax_bias table", true);
        if (table->dtype != in->dtype) fail(HPT_ERR_DTYPE, "softmax_bias table: dtype is %s, expected %s", dtype_name(table->dtype), dtype_name(in->dtype));
        if (table->ndim != 2 || table->shape[1] != s.heads) fail(HPT_ERR_SHAPE, "softmax_bias table: must be buckets x %lld heads", (long long)s.heads);
        a.buckets = make_buckets(table->shape[0], bidirectional != 0, max_distance);
        check_lengths(lengths, s, "softmax_bias lengths");
        check_workspace(workspace, "softmax_bias workspace");
        check_out(out, in->dtype, view_size(in), "softmax_bias output");
        Overlaps o{"softmax_bias"};
        o.reads(in, "the input");
        o.reads(table, "the table");
        o.reads(lengths, "the lengths");
        o.writes(out, in);
        if (workspace) {
            hpt_view w = *workspace;
            o.writes(&w);
        }
        if (view_size(in) == 0) return;
        a.x = in->data;
        a.matrices = r.kept;
        a.query_stride = in->strides[in->ndim - 2];
        a.table = table->data;
        a.table_bucket = table->strides[0];
        a.table_head = table->strides[1];
        a.out = out->data;
        a.lengths = lengths ? lengths->data : nullptr;
        a.lengths64 = lengths && lengths->dtype == HPT_I64;
        a.causal = causal != 0;
        a.heads = s.heads;
        a.queries = s.queries;
        a.rows = s.rows;
        a.keys = (int)s.keys;
        a.offset = query_offset;
        use_device(dev);
        hipStream_t st = (hipStream_t)stream;
        const int split = bias_split(in->dtype, s.rows, s.keys);
        with_workspace(dev, st, workspace, split > 1 ? (size_t)(s.rows * split) * 2 * sizeof(float) : 0, true, "softmax_bias", [&](void* p) {
            a.partial = (float*)p;
            a.split = p ? split : 1;
            launch_softmax_bias(in->dtype, a, st);
            check_launch("softmax_bias");
        });
    });
}

int32_t hpt_hip_softmax_bias_backward_workspace(const hpt_view* probs, int64_t buckets, size_t* bytes) {
    return guarded([&] {
        if (!bytes) fail(HPT_ERR_PARAM, "softmax_bias_backward_workspace: null output");
        const Scores s = scores_of(probs, "softmax_bias_backward probs");
        if (buckets < 2 || buckets > kMostBuckets) fail(HPT_ERR_PARAM, "position bias: %lld buckets, outside 2..%d", (long long)buckets, kMostBuckets);
        int per_item = 0;
        *bytes = s.rows * s.keys ? (size_t)(bias_grad_items(probs->dtype, s.batch * s.heads, s.queries, s.keys, &per_item) * buckets) * sizeof(float) : 0;
    });
}

int32_t hpt_hip_softmax_bias_backward(int32_t dev, void* stream, const hpt_view* probs, const hpt_view* grad, double scale,
                                      int32_t bidirectional, int64_t max_distance, int64_t query_offset, int32_t causal,
                                      const hpt_view* lengths, const hpt_view* workspace, hpt_view* grad_in, hpt_view* grad_table) {
    return guarded([&] {
        const Scores s = scores_of(probs, "softmax_bias_backward probs");
        const int64_t count = view_size(probs);
        if (s.keys >= kMostCols) fail(HPT_ERR_SHAPE, "softmax_bias_backward probs: rows of %lld elements, fewer than %lld expected", (long long)s.keys, (long long)kMostCols);
        BiasGradArgs a{};
        a.scale = check_bias_scale(scale, query_offset, "softmax_bias_backward");
        check_operand(probs, probs->dtype, count, nullptr, "softmax_bias_backward probs");
        check_operand(grad, probs->dtype, count, probs, "softmax_bias_backward grad");
        check_lengths(lengths, s, "softmax_bias_backward lengths");
        check_workspace(workspace, "softmax_bias_backward workspace");
        check_out(grad_in, probs->dtype, count, "softmax_bias_backward grad_in");
        int64_t buckets = 2;
        if (grad_table) {
            check_view(grad_table, "softmax_bias_backward grad_table", true);
            if (grad_table->ndim != 2 || grad_table->shape[1] != s.heads)
                fail(HPT_ERR_SHAPE, "softmax_bias_backward grad_table: must be buckets x %lld heads", (long long)s.heads);
            buckets = grad_table->shape[0];
            check_out(grad_table, HPT_F32, buckets * s.heads, "softmax_bias_backward grad_table");
        }
        // (without a table's gradient any buckets do: none of the results depends on them)
        a.buckets = grad_table ? make_buckets(buckets, bidirectional != 0, max_distance) : make_buckets(2, false, 2);
        Overlaps o{"softmax_bias_backward"};
        o.reads(probs, "the probabilities");
        o.reads(grad, "grad");
        o.reads(lengths, "the lengths");
        o.writes(grad_in, probs, grad);
        o.writes(grad_table);
        if (workspace) {
            hpt_view w = *workspace;
            o.writes(&w);
        }
        if (s.heads == 0 || (count == 0 && !grad_table)) return;
        a.p = probs->data;
        a.g = grad->data;
        a.out = grad_in->data;
        a.table_grad = grad_table ? (float*)grad_table->data : nullptr;
        a.lengths = lengths ? lengths->data : nullptr;
        a.lengths64 = lengths && lengths->dtype == HPT_I64;
        a.causal = causal != 0;
        a.heads = s.heads;
        a.queries = s.queries;
        a.rows = count ? s.rows : 0;
        a.keys = (int)s.keys;
        a.offset = query_offset;
        size_t bytes = 0;
        int per_item = 0;
        if (count && grad_table) bytes = (size_t)(bias_grad_items(probs->dtype, s.batch * s.heads, s.queries, s.keys, &per_item) * buckets) * sizeof(float);
        use_device(dev);
        hipStream_t st = (hipStream_t)stream;
        with_workspace(dev, st, workspace, bytes, false, "softmax_bias_backward", [&](void* p) {
            a.partial = (float*)p;
            launch_softmax_bias_backward(probs->dtype, a, st);
            check_launch("softmax_bias_backward");
        });
    });
}

int32_t hpt_hip_policy_loss_workspace(const hpt_view* logits, size_t* bytes) {
    return guarded([&] {
        if (!bytes) fail(HPT_ERR_PARAM, "policy_loss_workspace: null output");
        *bytes = policy_bytes(logits, logits_of(logits, "policy_loss logits"), true);
    });
}

int32_t hpt_hip_token_logp(int32_t dev, void* stream, const hpt_view* logits, const hpt_view* token, const hpt_view* workspace,
                           hpt_view* logp, hpt_view* lse) {
    return guarded([&] {
        const RowsOf r = logits_of(logits, "token_logp logits");
        check_tokens(token, r.rows, "token_logp token");
        check_workspace(workspace, "token_logp workspace");
        check_out(logp, HPT_F32, r.rows, "token_logp logp");
        check_out(lse, HPT_F32, r.rows, "token_logp lse");
        Overlaps o{"token_logp"};
        o.reads(logits, "the logits");
        o.reads(token, "the tokens");
        o.writes(logp);
        o.writes(lse);
        if (workspace) {
            hpt_view w = *workspace;
            o.writes(&w);
        }
        if (r.rows == 0) return;
        PolicyArgs a{};
        a.logp = (float*)logp->data;
        a.lse = (float*)lse->data;
        run_policy(dev, stream, logits, r, a, token, workspace, false, "token_logp");
    });
}

int32_t hpt_hip_policy_loss(int32_t dev, void* stream, const hpt_view* logits, const hpt_view* token, const hpt_view* old_logp,
                            const hpt_view* advantage, const hpt_view* reference, const hpt_view* mask, double clip_low,
                            double clip_high, double kl_weight, const hpt_view* workspace, hpt_view* loss, hpt_view* logp,
                            hpt_view* lse, hpt_view* weight) {
    return guarded([&] {
        const RowsOf r = logits_of(logits, "policy_loss logits");
        check_tokens(token, r.rows, "policy_loss token");
        check_operand(old_logp, HPT_F32, r.rows, nullptr, "policy_loss old_logp");
        check_operand(advantage, HPT_F32, r.rows, nullptr, "policy_loss advantage");
        if (reference) check_operand(reference, HPT_F32, r.rows, nullptr, "policy_loss reference");
        if (mask) {
            check_view(mask, "policy_loss mask", true);
            if (mask->dtype != HPT_F32 && mask->dtype != HPT_BOOL) fail(HPT_ERR_DTYPE, "policy_loss mask: dtype is %s, expected f32 or bool", dtype_name(mask->dtype));
            check_operand(mask, mask->dtype, r.rows, nullptr, "policy_loss mask");
        }
        if (!(clip_low >= 0 && clip_low <= 1) || !(clip_high >= 0 && clip_high <= 1e30)) fail(HPT_ERR_PARAM, "policy_loss: clip_low must be in 0..1 and clip_high not negative");
        if (!(std::abs(kl_weight) <= 1e30)) fail(HPT_ERR_PARAM, "policy_loss: kl_weight must be a finite number");
        if (kl_weight != 0 && !reference) fail(HPT_ERR_PARAM, "policy_loss: a KL term needs the reference's log-probabilities");
        check_workspace(workspace, "policy_loss workspace");
        check_out(loss, HPT_F32, 1, "policy_loss loss");
        check_out(logp, HPT_F32, r.rows, "policy_loss logp");
        check_out(lse, HPT_F32, r.rows, "policy_loss lse");
        check_out(weight, HPT_F32, r.rows, "policy_loss weight");
        Overlaps o{"policy_loss"};
        o.reads(logits, "the logits");
        o.reads(token, "the tokens");
        o.reads(old_logp, "old_logp");
        o.reads(advantage, "the advantages");
        o.reads(reference, "the reference");
        o.reads(mask, "the mask");
        o.writes(loss);
        o.writes(logp);
        o.writes(lse);
        o.writes(weight);
        if (workspace) {
            hpt_view w = *workspace;
            o.writes(&w);
        }
        PolicyArgs a{};
        a.old_logp = (const float*)old_logp->data;
        a.advantage = (const float*)advantage->data;
        a.reference = reference && kl_weight != 0 ? (const float*)reference->data : nullptr;
        a.mask = mask ? mask->data : nullptr;
        a.mask_bool = mask && mask->dtype == HPT_BOOL;
        a.clip_low = clip_low;
        a.clip_high = clip_high;
        a.kl_weight = kl_weight;
        a.loss = (float*)loss->data;
        a.logp = (float*)logp->data;
        a.lse = (float*)lse->data;
        a.weight = (float*)weight->data;
        run_policy(dev, stream, logits, r, a, token, workspace, true, "policy_loss");
    });
}

int32_t hpt_hip_policy_loss_backward(int32_t dev, void* stream, const hpt_view* logits, const hpt_view* token, const hpt_view* lse,
                                     const hpt_view* weight, double grad, hpt_view* grad_logits) {
    return guarded([&] {
        const RowsOf r = logits_of(logits, "policy_loss_backward logits");
        check_tokens(token, r.rows, "policy_loss_backward token");
        check_operand(lse, HPT_F32, r.rows, nullptr, "policy_loss_backward lse");
        check_operand(weight, HPT_F32, r.rows, nullptr, "policy_loss_backward weight");
        check_out(grad_logits, logits->dtype, view_size(logits), "policy_loss_backward grad_logits");
        Overlaps o{"policy_loss_backward"};
        o.reads(logits, "the logits");
        o.reads(token, "the tokens");
        o.reads(lse, "lse");
        o.reads(weight, "the weights");
        o.writes(grad_logits, logits);
        if (r.rows == 0) return;
        PolicyGradArgs a{};
        a.x = logits->data;
        a.kept = r.kept;
        a.token = token->data;
        a.token64 = token->dtype == HPT_I64;
        a.lse = (const float*)lse->data;
        a.weight = (const float*)weight->data;
        a.upstream = (float)grad;
        a.out = grad_logits->data;
        a.rows = r.rows;
        a.cols = (int)r.cols;
        use_device(dev);
        launch_policy_loss_backward(logits->dtype, a, (hipStream_t)stream);
        check_launch("policy_loss_backward");
    });
}

}  // extern "C"
