// dr_api.cpp -- the C ABI declared in include/dr_attn.h.
//
// Host-side bookkeeping only: argument validation with the reference's
// contract, device buffers, row metadata upload, launch planning.  All
// arithmetic on the attention path runs in the HIP kernels of the kernel
// sources beside it; there is no CPU fallback.  If no GPU is visible every
// compute entry point fails with DR_ERR_NO_DEVICE.
#include "dr_attn.h"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <limits>
#include <mutex>
#include <string>
#include <vector>

#include "dr_internal.hpp"

namespace {

thread_local std::string g_err;

// Every device and pinned host allocation the library makes goes through
// these two, which count it (dr_debug_alloc_count).
std::atomic<long> g_allocs{0};
template <typename T>
hipError_t dev_malloc(T** p, size_t bytes) {
    g_allocs.fetch_add(1, std::memory_order_relaxed);
    return hipMalloc(reinterpret_cast<void**>(p), bytes);
}
template <typename T>
hipError_t host_malloc(T** p, size_t bytes) {
    g_allocs.fetch_add(1, std::memory_order_relaxed);
    return hipHostMalloc(reinterpret_cast<void**>(p), bytes);
}

int fail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    g_err = buf;
    return code;
}

int hip_fail(hipError_t e, const char* what) {
    return fail(e == hipErrorOutOfMemory ? DR_ERR_OOM : DR_ERR_HIP, "%s: %s", what,
                hipGetErrorString(e));
}

#define DR_HIP(expr)                                    \
    do {                                                \
        hipError_t e_ = (expr);                         \
        if (e_ != hipSuccess) return hip_fail(e_, #expr); \
    } while (0)

#define DR_CHECK(expr)                 \
    do {                               \
        int rc_ = (expr);              \
        if (rc_ != DR_OK) return rc_;  \
    } while (0)

// Largest sequence position / window the kernels accept (int32 arithmetic
// on |qpos - kpos|).  The reference caps sequences at 32768 (model.rs:403-407).
constexpr size_t MAX_POS = (size_t)1 << 30;
// Row blocks (batch x kv head x 32-row group) whose key splits one call can
// merge in-kernel: the size of each context's ticket buffer.
constexpr size_t TICKETS = (size_t)1 << 16;
// Largest |scale| * sqrt(head_dim) a bf16 layer accepts unless a kernel
// family is forced (1 at the reference's usual 1/sqrt(head_dim)).
constexpr double MAX_BF16_SCALE = 2.0;

struct DevBuf {
    void* p = nullptr;
    size_t cap = 0;
};

int ensure(DevBuf& b, size_t bytes) {
    if (bytes <= b.cap) return DR_OK;
    if (b.p) {
        hipError_t e = hipFree(b.p);  // implicitly waits for work using it
        b.p = nullptr;
        b.cap = 0;
        if (e != hipSuccess) return hip_fail(e, "hipFree");
    }
    size_t nb = std::max(bytes, (size_t)4096);
    DR_HIP(dev_malloc(&b.p, nb));
    b.cap = nb;
    return DR_OK;
}

// The growing workspaces that kernel launches take (key-split partials, Q8_K
// activations).  A hipGraph captured on the context keeps the buffer pointer
// it was captured with, so a workspace is never freed or moved while the
// context lives: a larger request allocates a new buffer (at least twice the
// old size) and retires the old one, which dr_ctx_destroy frees.
int grow(DevBuf& b, size_t bytes, std::vector<void*>& retired) {
    if (bytes <= b.cap) return DR_OK;
    const size_t nb = std::max({bytes, 2 * b.cap, (size_t)4096});
    void* p = nullptr;
    DR_HIP(dev_malloc(&p, nb));
    if (b.p) retired.push_back(b.p);
    b.p = p;
    b.cap = nb;
    return DR_OK;
}

void release(DevBuf& b) {
    if (b.p) (void)hipFree(b.p);
    b.p = nullptr;
    b.cap = 0;
}

int hd_tile_for(size_t hd) { return hd <= 64 ? 64 : (hd <= 128 ? 128 : (hd <= 256 ? 256 : 512)); }

size_t round_up(size_t x, size_t m) { return (x + m - 1) / m * m; }

}  // namespace

struct dr_ctx {
    int device = 0;
    hipStream_t stream = nullptr;
    hipStream_t own = nullptr;
    int n_cu = 0;
    int force_split = 0;
    int force_rb = 0;
    int force_kq = 0;
    int force_rows = 0;  // query rows per compute wave (0: automatic)
    int force_kernel = 0;  // dr::KernelKind (0: automatic)
    int q_bf16 = 0;        // the cached entry points' Q rows are bf16
    int o_bf16 = 0;        // the cached entry points write bf16 output rows
    int merge_in_kernel = 1;  // key splits of the per-wave-stream kernel merge in-kernel
    dr::LaunchPlan last{};
    bool has_last = false;
    DevBuf part;                         // key-split partials (grow() only)
    DevBuf q, k, v, kc, vtc, meta, out;  // dr_attention() staging
    DevBuf kclo, vtclo;                  // dr_attention(): lo halves of K and V^T
    DevBuf q8k;                          // dr_qmatmul's Q8_K activations (grow() only)
    DevBuf qpre;                         // hi/lo attention: Q after its epilogue (grow() only)
    DevBuf tick;                         // in-kernel split merge: per-row-block tickets, zero at rest
    std::vector<void*> retired;          // workspaces replaced by larger ones
    // dr_ctx_destroy's reference plus one per pass, cache and RoPE table made
    // on the context: it is freed when the last of them is destroyed, so the
    // objects that use it may be destroyed before or after it
    std::atomic<int> refs{1};
    // set while a host thread is inside an entry point that uses the
    // context's workspaces, tickets or launch record (CtxUse)
    std::atomic<bool> busy{false};
    // dr_ctx_set_stream: the new stream waits on this, recorded on the old one
    hipEvent_t switch_ev = nullptr;
};

struct dr_pass {
    dr_ctx* ctx = nullptr;
    int* d_pos = nullptr;
    size_t n = 0;
    size_t cap = 0;
    size_t min_pos = 0, max_pos = 0;
};

struct dr_rope {
    dr_ctx* ctx = nullptr;
    size_t max_len = 0, rope_dim = 0;
    float* d_table = nullptr;  // [max_len][rope_dim/2][2] (sin, cos)
};

struct dr_step_cache {
    struct Slot {
        // split_active's state (cache.rs:31-34).  It lives on the host, or,
        // once a device-side call has used it, in d_prev / d_lc until a host
        // call takes it back (dev_state says which copy is current).
        std::vector<int32_t> prev_seq, last_changed;
        int32_t* d_prev = nullptr;
        int32_t* d_lc = nullptr;
        bool dev_state = false;
        bool initialized = false;
        size_t vicinity = 0;
    };
    dr_ctx* ctx = nullptr;
    size_t n_total = 0, cap = 0, n_layer = 0, n_batch = 0;
    std::vector<int> hkv, hd, hd_tile;
    std::vector<uint16_t*> k, vt;  // [layer * n_batch + batch]
    std::vector<uint16_t*> klo, vlo;  // lo halves of K and V^T (DR_PRECISION_HILO layers), else nullptr
    // DR_PRECISION_FP8 layers: code planes and scale bytes (then k, vt, klo and vlo are nullptr), else nullptr
    std::vector<uint8_t*> k8, v8, sc;
    std::vector<Slot> slot;
    int32_t* h_meta = nullptr;     // [6] split results, pinned host memory the kernel writes
    int32_t* h_meta_dev = nullptr; // its device address
};

namespace {

int use_device(const dr_ctx* ctx) {
    DR_HIP(hipSetDevice(ctx->device));
    return DR_OK;
}

// Capacity for n positions in a pass's device array (contents not kept).
int reserve_pass(dr_pass* p, size_t n) {
    if (n <= p->cap) return DR_OK;
    DR_CHECK(use_device(p->ctx));
    if (p->d_pos) {
        hipError_t e = hipFree(p->d_pos);
        p->d_pos = nullptr;
        p->cap = 0;
        if (e != hipSuccess) return hip_fail(e, "hipFree");
    }
    DR_HIP(dev_malloc(&p->d_pos, n * sizeof(int32_t)));
    p->cap = n;
    return DR_OK;
}

int upload_pass(dr_pass* p, const size_t* active, size_t n) {
    if (n > 0 && !active) return fail(DR_ERR_INVALID, "pass: active is NULL with n_active=%zu", n);
    std::vector<int32_t> h(n);
    size_t mx = 0;
    for (size_t i = 0; i < n; ++i) {
        if (active[i] >= MAX_POS)
            return fail(DR_ERR_INVALID, "pass: position %zu exceeds %zu", active[i], MAX_POS);
        if (i > 0 && active[i] <= active[i - 1])
            return fail(DR_ERR_INVALID, "pass: positions must be strictly ascending (index %zu)", i);
        h[i] = (int32_t)active[i];
        mx = std::max(mx, active[i]);
    }
    DR_CHECK(use_device(p->ctx));
    DR_CHECK(reserve_pass(p, n));
    if (n > 0) {
        DR_HIP(hipMemcpyAsync(p->d_pos, h.data(), n * sizeof(int32_t), hipMemcpyHostToDevice,
                              p->ctx->stream));
        DR_HIP(hipStreamSynchronize(p->ctx->stream));
    }
    p->n = n;
    p->min_pos = n > 0 ? active[0] : 0;
    p->max_pos = mx;
    return DR_OK;
}

std::mutex g_default_mu;
dr_ctx* g_default_ctx = nullptr;

// One host thread at a time per context: an entry point that uses the
// context's workspaces, split tickets or launch record holds this for the
// call, and a second thread that arrives meanwhile gets DR_ERR_BUSY instead
// of racing on them.
class CtxUse {
  public:
    explicit CtxUse(dr_ctx* c) : c_(c), ok_(!c->busy.exchange(true, std::memory_order_acquire)) {}
    ~CtxUse() {
        if (ok_) c_->busy.store(false, std::memory_order_release);
    }
    CtxUse(const CtxUse&) = delete;
    CtxUse& operator=(const CtxUse&) = delete;
    bool ok() const { return ok_; }

  private:
    dr_ctx* c_;
    bool ok_;
};

#define DR_CTX_USE(ctx, who)                                                                          \
    CtxUse ctx_use_(ctx);                                                                             \
    if (!ctx_use_.ok())                                                                               \
        return fail(DR_ERR_BUSY, "%s: the context is in use by another thread (one thread at a time)", \
                    who)

bool capturing(hipStream_t st) {
    hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
    return hipStreamIsCapturing(st, &cs) == hipSuccess && cs != hipStreamCaptureStatusNone;
}

// dr_attention_cached_noalloc's device scratch is one array per GPU, shared
// by every context: a call on another stream than the previous call on that
// GPU first waits (on the device) for the previous call's kernels, so two
// calls never use it at once.  The event is made at dr_ctx_create, so the
// call itself creates nothing.
struct ScratchOrder {
    std::mutex mu;
    hipEvent_t done = nullptr;   // recorded after each call's launches
    hipStream_t last = nullptr;  // the stream of the previous call
};
ScratchOrder g_scratch_order[64];

}  // namespace

extern "C" {

const char* dr_last_error(void) { return g_err.c_str(); }

const char* dr_version(void) { return "0.1.0"; }

int dr_device_count(void) {
    int n = 0;
    if (hipGetDeviceCount(&n) != hipSuccess) {
        (void)hipGetLastError();
        return 0;
    }
    return n;
}

int dr_ctx_create(int device, dr_ctx** out) {
    if (!out) return fail(DR_ERR_INVALID, "dr_ctx_create: out is NULL");
    *out = nullptr;
    const int n = dr_device_count();
    if (n <= 0) return fail(DR_ERR_NO_DEVICE, "no HIP device visible");
    if (device < 0 || device >= n)
        return fail(DR_ERR_INVALID, "device %d out of range (%d visible)", device, n);
    DR_HIP(hipSetDevice(device));
    dr_ctx* c = new dr_ctx();
    c->device = device;
    hipError_t e = hipStreamCreateWithFlags(&c->own, hipStreamNonBlocking);
    if (e != hipSuccess) {
        delete c;
        return hip_fail(e, "hipStreamCreateWithFlags");
    }
    c->stream = c->own;
    // this device's address of the fixed scratch (dr_attention_cached_noalloc)
    e = dr::scratch_init(device);
    if (e != hipSuccess) {
        (void)hipStreamDestroy(c->own);
        delete c;
        return hip_fail(e, "hipGetSymbolAddress(scratch)");
    }
    e = hipEventCreateWithFlags(&c->switch_ev, hipEventDisableTiming);
    if (e == hipSuccess && device < 64) {
        ScratchOrder& so = g_scratch_order[device];
        std::lock_guard<std::mutex> lk(so.mu);
        if (!so.done) e = hipEventCreateWithFlags(&so.done, hipEventDisableTiming);
    }
    if (e != hipSuccess) {
        if (c->switch_ev) (void)hipEventDestroy(c->switch_ev);
        (void)hipStreamDestroy(c->own);
        delete c;
        return hip_fail(e, "hipEventCreateWithFlags");
    }
    e = hipDeviceGetAttribute(&c->n_cu, hipDeviceAttributeMultiprocessorCount, device);
    if (e != hipSuccess) {
        (void)hipEventDestroy(c->switch_ev);
        (void)hipStreamDestroy(c->own);
        delete c;
        return hip_fail(e, "hipDeviceGetAttribute");
    }
    // the in-kernel split merge's tickets: allocated and zeroed here, once,
    // so that no call allocates or clears them (each merge resets its own)
    e = dev_malloc(&c->tick.p, TICKETS * sizeof(int));
    if (e == hipSuccess) {
        c->tick.cap = TICKETS * sizeof(int);
        e = hipMemsetAsync(c->tick.p, 0, TICKETS * sizeof(int), c->own);
        if (e == hipSuccess) e = hipStreamSynchronize(c->own);
    }
    if (e != hipSuccess) {
        release(c->tick);
        (void)hipEventDestroy(c->switch_ev);
        (void)hipStreamDestroy(c->own);
        delete c;
        return hip_fail(e, "ticket buffer");
    }
    *out = c;
    return DR_OK;
}

int dr_ctx_set_stream(dr_ctx* ctx, void* stream) {
    if (!ctx) return fail(DR_ERR_INVALID, "dr_ctx_set_stream: ctx is NULL");
    DR_CTX_USE(ctx, "dr_ctx_set_stream");
    hipStream_t ns = stream ? static_cast<hipStream_t>(stream) : ctx->own;
    if (ns != ctx->stream && !capturing(ctx->stream) && !capturing(ns)) {
        // the new stream starts after the work already queued on the old one,
        // so the context's workspaces and split tickets are never in use on
        // both (a stream under graph capture is ordered by its graph instead)
        DR_CHECK(use_device(ctx));
        DR_HIP(hipEventRecord(ctx->switch_ev, ctx->stream));
        DR_HIP(hipStreamWaitEvent(ns, ctx->switch_ev, 0));
    }
    ctx->stream = ns;
    return DR_OK;
}

void* dr_ctx_stream(dr_ctx* ctx) { return ctx ? static_cast<void*>(ctx->stream) : nullptr; }

int dr_ctx_synchronize(dr_ctx* ctx) {
    if (!ctx) return fail(DR_ERR_INVALID, "dr_ctx_synchronize: ctx is NULL");
    DR_CHECK(use_device(ctx));
    DR_HIP(hipStreamSynchronize(ctx->stream));
    return DR_OK;
}

namespace {

void ctx_free(dr_ctx* ctx) {
    (void)hipSetDevice(ctx->device);
    if (ctx->stream) (void)hipStreamSynchronize(ctx->stream);
    for (DevBuf* b : {&ctx->part, &ctx->q, &ctx->k, &ctx->v, &ctx->kc, &ctx->vtc, &ctx->kclo, &ctx->vtclo,
                      &ctx->meta, &ctx->out, &ctx->q8k, &ctx->qpre, &ctx->tick})
        release(*b);
    for (void* p : ctx->retired) (void)hipFree(p);
    if (ctx->own) (void)hipStreamDestroy(ctx->own);
    if (ctx->switch_ev) (void)hipEventDestroy(ctx->switch_ev);
    delete ctx;
}

}  // namespace

static void ctx_retain(dr_ctx* ctx) { ctx->refs.fetch_add(1, std::memory_order_relaxed); }

static void ctx_release(dr_ctx* ctx) {
    if (ctx->refs.fetch_sub(1, std::memory_order_acq_rel) == 1) ctx_free(ctx);
}

void dr_ctx_destroy(dr_ctx* ctx) {
    if (ctx) ctx_release(ctx);
}

int dr_ctx_last_launch(const dr_ctx* ctx, dr_launch_info* info) {
    if (!ctx || !info) return fail(DR_ERR_INVALID, "dr_ctx_last_launch: NULL argument");
    if (!ctx->has_last) return fail(DR_ERR_INVALID, "no attention launched on this context yet");
    info->n_split = ctx->last.n_split;
    info->n_workgroups = ctx->last.n_workgroups;
    info->waves_per_wg = ctx->last.waves;
    info->block_n = ctx->last.block_n;
    info->head_dim_tile = ctx->last.hd_tile;
    info->row_blocks = ctx->last.rb;
    info->key_groups = ctx->last.kq;
    info->rows_per_wave = ctx->last.w16 ? 16 : 32;
    info->kernel = ctx->last.kernel;
    info->split_merge = ctx->last.merge;
    return DR_OK;
}

int dr_ctx_set_split(dr_ctx* ctx, int n_split) {
    if (!ctx) return fail(DR_ERR_INVALID, "dr_ctx_set_split: ctx is NULL");
    if (n_split < 0 || n_split > 64) return fail(DR_ERR_INVALID, "n_split %d not in 0..64", n_split);
    ctx->force_split = n_split;
    return DR_OK;
}

int dr_ctx_set_wave_rows(dr_ctx* ctx, int rows) {
    if (!ctx) return fail(DR_ERR_INVALID, "dr_ctx_set_wave_rows: ctx is NULL");
    if (rows != 0 && rows != 16 && rows != 32) return fail(DR_ERR_INVALID, "rows %d not 0, 16 or 32", rows);
    ctx->force_rows = rows;
    return DR_OK;
}

int dr_ctx_set_kernel(dr_ctx* ctx, int kernel) {
    if (!ctx) return fail(DR_ERR_INVALID, "dr_ctx_set_kernel: ctx is NULL");
    if (kernel < DR_KERNEL_AUTO || kernel > DR_KERNEL_FP8)
        return fail(DR_ERR_INVALID, "kernel %d not DR_KERNEL_AUTO, _STAGED, _STREAMS, _HILO or _FP8", kernel);
    ctx->force_kernel = kernel;
    return DR_OK;
}

int dr_ctx_set_q_dtype(dr_ctx* ctx, int dtype) {
    if (!ctx) return fail(DR_ERR_INVALID, "dr_ctx_set_q_dtype: ctx is NULL");
    if (dtype != DR_DTYPE_F32 && dtype != DR_DTYPE_BF16)
        return fail(DR_ERR_INVALID, "dtype %d not DR_DTYPE_F32 or DR_DTYPE_BF16", dtype);
    ctx->q_bf16 = dtype == DR_DTYPE_BF16 ? 1 : 0;
    return DR_OK;
}

int dr_ctx_set_o_dtype(dr_ctx* ctx, int dtype) {
    if (!ctx) return fail(DR_ERR_INVALID, "dr_ctx_set_o_dtype: ctx is NULL");
    if (dtype != DR_DTYPE_F32 && dtype != DR_DTYPE_BF16)
        return fail(DR_ERR_INVALID, "dtype %d not DR_DTYPE_F32 or DR_DTYPE_BF16", dtype);
    ctx->o_bf16 = dtype == DR_DTYPE_BF16 ? 1 : 0;
    return DR_OK;
}

int dr_ctx_set_split_merge(dr_ctx* ctx, int in_kernel) {
    if (!ctx) return fail(DR_ERR_INVALID, "dr_ctx_set_split_merge: ctx is NULL");
    if (in_kernel != 0 && in_kernel != 1) return fail(DR_ERR_INVALID, "in_kernel %d not 0 or 1", in_kernel);
    ctx->merge_in_kernel = in_kernel;
    return DR_OK;
}

int dr_ctx_set_tuning(dr_ctx* ctx, int row_blocks, int key_groups, int n_split) {
    if (!ctx) return fail(DR_ERR_INVALID, "dr_ctx_set_tuning: ctx is NULL");
    if (row_blocks < 0 || row_blocks > 8 || key_groups < 0 || key_groups > 8)
        return fail(DR_ERR_INVALID, "row_blocks/key_groups not in 0..8");
    DR_CHECK(dr_ctx_set_split(ctx, n_split));
    ctx->force_rb = row_blocks;
    ctx->force_kq = key_groups;
    return DR_OK;
}

// ---------------------------------------------------------------- passes

int dr_pass_create(dr_ctx* ctx, const size_t* active, size_t n_active, dr_pass** out) {
    if (!ctx || !out) return fail(DR_ERR_INVALID, "dr_pass_create: NULL argument");
    *out = nullptr;
    dr_pass* p = new dr_pass();
    p->ctx = ctx;
    ctx_retain(ctx);
    int rc = upload_pass(p, active, n_active);
    if (rc != DR_OK) {
        dr_pass_destroy(p);
        return rc;
    }
    *out = p;
    return DR_OK;
}

int dr_pass_set(dr_pass* pass, const size_t* active, size_t n_active) {
    if (!pass) return fail(DR_ERR_INVALID, "dr_pass_set: pass is NULL");
    return upload_pass(pass, active, n_active);
}

size_t dr_pass_len(const dr_pass* pass) { return pass ? pass->n : 0; }

int dr_pass_positions(const dr_pass* pass, size_t* out, size_t cap) {
    if (!pass) return fail(DR_ERR_INVALID, "dr_pass_positions: pass is NULL");
    if (cap < pass->n) return fail(DR_ERR_INVALID, "dr_pass_positions: cap %zu < %zu", cap, pass->n);
    if (pass->n == 0) return DR_OK;
    if (!out) return fail(DR_ERR_INVALID, "dr_pass_positions: out is NULL");
    DR_CHECK(use_device(pass->ctx));
    std::vector<int32_t> h(pass->n);
    DR_HIP(hipMemcpyAsync(h.data(), pass->d_pos, pass->n * sizeof(int32_t), hipMemcpyDeviceToHost,
                          pass->ctx->stream));
    DR_HIP(hipStreamSynchronize(pass->ctx->stream));
    for (size_t i = 0; i < pass->n; ++i) out[i] = (size_t)h[i];
    return DR_OK;
}

void dr_pass_destroy(dr_pass* pass) {
    if (!pass) return;
    dr_ctx* ctx = pass->ctx;
    if (pass->d_pos) {
        (void)hipSetDevice(ctx->device);
        (void)hipStreamSynchronize(ctx->stream);
        (void)hipFree(pass->d_pos);
    }
    delete pass;
    ctx_release(ctx);
}

// ---------------------------------------------------------------- cache

extern "C++" {
namespace {

bool precision_ok(int precision) {
    return precision == DR_PRECISION_BF16 || precision == DR_PRECISION_HILO || precision == DR_PRECISION_FP8;
}

// The planes that a layer of some precision keeps per batch slot, and where
// each is held; bytes of one of them.
struct Plane {
    std::vector<uint16_t*>* p16;
    std::vector<uint8_t*>* p8;
    size_t bytes;
    void* get(size_t i) const { return p16 ? static_cast<void*>((*p16)[i]) : (*p8)[i]; }
    void set(size_t i, void* p) const {
        if (p16)
            (*p16)[i] = static_cast<uint16_t*>(p);
        else
            (*p8)[i] = static_cast<uint8_t*>(p);
    }
};

std::vector<Plane> planes_of(dr_step_cache* c, size_t layer, int precision) {
    const size_t values = (size_t)c->hkv[layer] * c->cap * c->hd_tile[layer];
    if (precision == DR_PRECISION_FP8)
        return {{nullptr, &c->k8, values},
                {nullptr, &c->v8, values},
                {nullptr, &c->sc, (size_t)c->hkv[layer] * c->cap * 2}};
    std::vector<Plane> v = {{&c->k, nullptr, 2 * values}, {&c->vt, nullptr, 2 * values}};
    if (precision == DR_PRECISION_HILO) {
        v.push_back({&c->klo, nullptr, 2 * values});
        v.push_back({&c->vlo, nullptr, 2 * values});
    }
    return v;
}

// Allocates (zeroed) what of a layer's planes for `precision` is not there
// yet.  On failure what this call allocated is freed again.
int add_planes(dr_step_cache* c, size_t layer, int precision, const char* what) {
    std::vector<std::pair<Plane, size_t>> made;
    hipError_t e = hipSuccess;
    for (const Plane& pl : planes_of(c, layer, precision))
        for (size_t i = layer * c->n_batch; e == hipSuccess && i < (layer + 1) * c->n_batch; ++i) {
            if (pl.get(i)) continue;
            void* p = nullptr;
            e = dev_malloc(&p, pl.bytes);
            if (e != hipSuccess) break;
            pl.set(i, p);
            made.push_back({pl, i});
            // (on the context's own stream and waited for: its calls run on
            // streams that the null stream does not order)
            e = hipMemsetAsync(p, 0, pl.bytes, c->ctx->own);
        }
    if (e == hipSuccess) e = hipStreamSynchronize(c->ctx->own);
    if (e == hipSuccess) return DR_OK;
    for (auto& m : made) {
        (void)hipFree(m.first.get(m.second));
        m.first.set(m.second, nullptr);
    }
    return hip_fail(e, what);
}

int create_cache(dr_ctx* ctx, size_t n_total, size_t n_layer, const size_t* n_head_kv, const size_t* head_dim,
                 const int* precision, size_t n_batch, dr_step_cache** out) {
    if (!ctx || !out) return fail(DR_ERR_INVALID, "dr_cache_create: NULL argument");
    *out = nullptr;
    if (n_layer > 0 && (!n_head_kv || !head_dim))
        return fail(DR_ERR_INVALID, "dr_cache_create: per-layer arrays are NULL");
    if (n_batch < 1 || n_batch > (size_t)dr::MAX_BATCH)
        return fail(DR_ERR_INVALID, "n_batch %zu not in 1..%d", n_batch, dr::MAX_BATCH);
    if (n_total >= MAX_POS) return fail(DR_ERR_INVALID, "n_total %zu too large", n_total);
    for (size_t l = 0; l < n_layer; ++l) {
        if (n_head_kv[l] < 1 || n_head_kv[l] > 4096)
            return fail(DR_ERR_INVALID, "layer %zu: n_head_kv %zu invalid", l, n_head_kv[l]);
        if (head_dim[l] < 1) return fail(DR_ERR_INVALID, "layer %zu: head_dim is 0", l);
        if (head_dim[l] > 512)
            return fail(DR_ERR_UNSUPPORTED, "layer %zu: head_dim %zu > 512 not built", l,
                        head_dim[l]);
    }
    DR_CHECK(use_device(ctx));
    dr_step_cache* c = new dr_step_cache();
    c->ctx = ctx;
    ctx_retain(ctx);
    c->n_total = n_total;
    c->cap = round_up(std::max(n_total, (size_t)1), dr::KEY_ALIGN);
    c->n_layer = n_layer;
    c->n_batch = n_batch;
    for (auto* v : {&c->k, &c->vt, &c->klo, &c->vlo}) v->assign(n_layer * n_batch, nullptr);
    for (auto* v : {&c->k8, &c->v8, &c->sc}) v->assign(n_layer * n_batch, nullptr);
    c->slot.resize(n_batch);
    for (auto& s : c->slot) {
        s.prev_seq.assign(n_total, -1);
        s.last_changed.assign(n_total, -1);
    }
    for (size_t l = 0; l < n_layer; ++l) {
        c->hkv.push_back((int)n_head_kv[l]);
        c->hd.push_back((int)head_dim[l]);
        c->hd_tile.push_back(hd_tile_for(head_dim[l]));
    }
    for (size_t l = 0; l < n_layer; ++l) {
        const int rc = add_planes(c, l, precision ? precision[l] : DR_PRECISION_BF16, "KV cache allocation");
        if (rc != DR_OK) {
            const std::string msg = g_err;
            dr_cache_destroy(c);
            return fail(rc, "%s", msg.c_str());
        }
    }
    *out = c;
    return DR_OK;
}

}  // namespace
}  // extern "C++"

int dr_cache_create(dr_ctx* ctx, size_t n_total, size_t n_layer, const size_t* n_head_kv,
                    const size_t* head_dim, size_t n_batch, dr_step_cache** out) {
    return create_cache(ctx, n_total, n_layer, n_head_kv, head_dim, nullptr, n_batch, out);
}

int dr_cache_create_layers(dr_ctx* ctx, size_t n_total, size_t n_layer, const size_t* n_head_kv,
                           const size_t* head_dim, const int* precision, size_t n_batch,
                           dr_step_cache** out) {
    if (precision)
        for (size_t l = 0; l < n_layer; ++l)
            if (!precision_ok(precision[l]))
                return fail(DR_ERR_INVALID, "layer %zu: precision %d not DR_PRECISION_BF16, _HILO or _FP8", l,
                            precision[l]);
    return create_cache(ctx, n_total, n_layer, n_head_kv, head_dim, precision, n_batch, out);
}

void dr_cache_destroy(dr_step_cache* cache) {
    if (!cache) return;
    (void)hipSetDevice(cache->ctx->device);
    (void)hipStreamSynchronize(cache->ctx->stream);
    for (auto* v : {&cache->k, &cache->vt, &cache->klo, &cache->vlo})
        for (uint16_t* p : *v)
            if (p) (void)hipFree(p);
    for (auto* v : {&cache->k8, &cache->v8, &cache->sc})
        for (uint8_t* p : *v)
            if (p) (void)hipFree(p);
    for (auto& s : cache->slot) {
        if (s.d_prev) (void)hipFree(s.d_prev);
        if (s.d_lc) (void)hipFree(s.d_lc);
    }
    if (cache->h_meta) (void)hipHostFree(cache->h_meta);
    dr_ctx* ctx = cache->ctx;
    delete cache;
    ctx_release(ctx);
}

int dr_cache_set_precision(dr_step_cache* cache, size_t layer, int precision) {
    if (!cache) return fail(DR_ERR_INVALID, "dr_cache_set_precision: cache is NULL");
    if (layer >= cache->n_layer)
        return fail(DR_ERR_INVALID, "dr_cache_set_precision: layer %zu >= %zu", layer, cache->n_layer);
    if (!precision_ok(precision))
        return fail(DR_ERR_INVALID, "dr_cache_set_precision: precision %d is not DR_PRECISION_BF16 (0), "
                    "DR_PRECISION_HILO (1) or DR_PRECISION_FP8 (2)", precision);
    const std::vector<Plane> keep = planes_of(cache, layer, precision);
    std::vector<Plane> drop;
    for (int other : {DR_PRECISION_HILO, DR_PRECISION_FP8})
        for (const Plane& pl : planes_of(cache, layer, other)) {
            bool kept = false;
            for (const Plane& k : keep) kept = kept || (k.p16 == pl.p16 && k.p8 == pl.p8);
            if (!kept) drop.push_back(pl);
        }
    const size_t first = layer * cache->n_batch, last = first + cache->n_batch;
    bool same = true;
    for (size_t i = first; i < last; ++i) {
        for (const Plane& pl : keep) same = same && pl.get(i);
        for (const Plane& pl : drop) same = same && !pl.get(i);
    }
    if (same) return DR_OK;  // (nothing asked of the device: a stream may be under capture)
    if (capturing(cache->ctx->stream) || capturing(cache->ctx->own))
        return fail(DR_ERR_INVALID, "dr_cache_set_precision: the context's stream is under graph capture (a graph "
                    "would keep planes that this call frees)");
    DR_CHECK(use_device(cache->ctx));
    // (zero: rows stored before this call carry no lo half, and none of them
    // passes between the 8 bit planes and the others)
    DR_CHECK(add_planes(cache, layer, precision, "cache plane allocation"));
    bool waited = false;
    for (const Plane& pl : drop)
        for (size_t i = first; i < last; ++i) {
            if (!pl.get(i)) continue;
            if (!waited) (void)hipStreamSynchronize(cache->ctx->stream);
            waited = true;
            (void)hipFree(pl.get(i));
            pl.set(i, nullptr);
        }
    return DR_OK;
}

// ---------------------------------------------------------------- Q/K/V epilogue


int dr_rope_create(dr_ctx* ctx, size_t max_len, size_t rope_dim, float theta,
                   const float* freq_factors, dr_rope** out) {
    if (!ctx || !out) return fail(DR_ERR_INVALID, "dr_rope_create: NULL argument");
    *out = nullptr;
    if (rope_dim < 2 || rope_dim % 2 != 0 || rope_dim > 512)
        return fail(DR_ERR_INVALID, "dr_rope_create: rope_dim %zu not even in 2..512", rope_dim);
    if (max_len < 1 || max_len > ((size_t)1 << 27) / rope_dim)
        return fail(DR_ERR_INVALID, "dr_rope_create: max_len %zu not in 1..%zu", max_len,
                    ((size_t)1 << 27) / rope_dim);
    // build_rope_cache_ff (ops.rs:396-417), in f32 like Rust's f32::powf /
    // sin / cos (libm powf / sinf / cosf)
    const size_t half = rope_dim / 2;
    std::vector<float> h(max_len * half * 2);
    for (size_t t = 0; t < max_len; ++t)
        for (size_t i = 0; i < half; ++i) {
            const float e = 2.0f * (float)i / (float)rope_dim;
            float freq = 1.0f / powf(theta, e);
            if (freq_factors) freq /= freq_factors[i];
            const float ang = (float)t * freq;
            h[(t * half + i) * 2] = sinf(ang);
            h[(t * half + i) * 2 + 1] = cosf(ang);
        }
    DR_CHECK(use_device(ctx));
    dr_rope* r = new dr_rope();
    r->ctx = ctx;
    ctx_retain(ctx);
    r->max_len = max_len;
    r->rope_dim = rope_dim;
    hipError_t e = dev_malloc(reinterpret_cast<void**>(&r->d_table), h.size() * sizeof(float));
    if (e == hipSuccess)
        e = hipMemcpy(r->d_table, h.data(), h.size() * sizeof(float), hipMemcpyHostToDevice);
    if (e != hipSuccess) {
        dr_rope_destroy(r);
        return hip_fail(e, "RoPE table");
    }
    *out = r;
    return DR_OK;
}

void dr_rope_destroy(dr_rope* rope) {
    if (!rope) return;
    (void)hipSetDevice(rope->ctx->device);
    (void)hipStreamSynchronize(rope->ctx->stream);
    if (rope->d_table) (void)hipFree(rope->d_table);
    dr_ctx* ctx = rope->ctx;
    delete rope;
    ctx_release(ctx);
}

int dr_qkv_epilogue(dr_ctx* ctx, const dr_pass* pass, float* q, float* k, float* v, size_t n_head,
                    size_t n_head_kv, size_t head_dim, const float* bq, const float* bk,
                    const float* bv, const float* q_norm_w, const float* k_norm_w, int v_norm,
                    float eps, const dr_rope* rope) {
    if (!ctx || !pass) return fail(DR_ERR_INVALID, "dr_qkv_epilogue: ctx/pass is NULL");
    if (pass->ctx != ctx) return fail(DR_ERR_INVALID, "dr_qkv_epilogue: pass uses another context");
    if (head_dim < 1 || head_dim > 512)
        return fail(DR_ERR_UNSUPPORTED, "dr_qkv_epilogue: head_dim %zu not in 1..512", head_dim);
    if (n_head_kv == 0 || n_head % n_head_kv != 0)
        return fail(DR_ERR_INVALID, "n_head %zu is not a multiple of n_head_kv %zu", n_head, n_head_kv);
    if (rope) {
        if (rope->ctx != ctx) return fail(DR_ERR_INVALID, "dr_qkv_epilogue: rope uses another context");
        if (rope->rope_dim > head_dim)
            return fail(DR_ERR_INVALID, "rope_dim %zu > head_dim %zu", rope->rope_dim, head_dim);
        if (pass->n > 0 && pass->max_pos >= rope->max_len)
            return fail(DR_ERR_INVALID, "position %zu >= the RoPE table's %zu", pass->max_pos,
                        rope->max_len);
    }
    if (pass->n == 0) return DR_OK;
    if (!q || !k || !v) return fail(DR_ERR_INVALID, "dr_qkv_epilogue: q/k/v is NULL");
    if (pass->n * (n_head + 2 * n_head_kv) >= (size_t)1 << 31)
        return fail(DR_ERR_INVALID, "dr_qkv_epilogue: %zu rows x %zu heads is too many", pass->n,
                    n_head + 2 * n_head_kv);
    DR_CHECK(use_device(ctx));
    dr::EpiArgs a{};
    a.q = q;
    a.k = k;
    a.v = v;
    a.pos = pass->d_pos;
    a.pos0 = pass->n > 0 && pass->max_pos - pass->min_pos + 1 == pass->n ? (int)pass->min_pos : -1;
    a.n = (int)pass->n;
    a.n_head = (int)n_head;
    a.n_head_kv = (int)n_head_kv;
    a.hd = (int)head_dim;
    a.bq = bq;
    a.bk = bk;
    a.bv = bv;
    a.qn_w = q_norm_w;
    a.kn_w = k_norm_w;
    a.v_norm = v_norm ? 1 : 0;
    a.eps = eps;
    a.rope = rope ? rope->d_table : nullptr;
    a.rot = rope ? (int)rope->rope_dim : 0;
    a.vec = head_dim % 4 == 0 && (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) & 15) == 0;
    hipError_t e = dr::launch_epilogue(a, ctx->stream);
    if (e != hipSuccess) return hip_fail(e, "qkv_epilogue launch");
    return DR_OK;
}

static int check_slot(const dr_step_cache* c, size_t layer, size_t batch, const char* who) {
    if (!c) return fail(DR_ERR_INVALID, "%s: cache is NULL", who);
    if (layer >= c->n_layer) return fail(DR_ERR_INVALID, "%s: layer %zu >= %zu", who, layer, c->n_layer);
    if (batch >= c->n_batch) return fail(DR_ERR_INVALID, "%s: batch %zu >= %zu", who, batch, c->n_batch);
    return DR_OK;
}

// StepCache::store (cache.rs:62-71) of a pass's rows, with the K / V part of
// the Q/K/V epilogue (forward.rs:291-310) applied on the way when asked.
static int store_rows(dr_step_cache* cache, size_t layer, size_t batch, const dr_pass* pass,
                      const float* k, const float* v, const float* k_norm_w, float eps,
                      const float* kb, const float* vb, int v_norm, const dr_rope* rope,
                      size_t kv_stride = 0);

int dr_cache_store(dr_step_cache* cache, size_t layer, size_t batch, const dr_pass* pass,
                   const float* k, const float* v, const float* k_norm_w, float eps) {
    return store_rows(cache, layer, batch, pass, k, v, k_norm_w, eps, nullptr, nullptr, 0, nullptr);
}

static int store_rows(dr_step_cache* cache, size_t layer, size_t batch, const dr_pass* pass,
                      const float* k, const float* v, const float* k_norm_w, float eps,
                      const float* kb, const float* vb, int v_norm, const dr_rope* rope,
                      size_t kv_stride) {
    DR_CHECK(check_slot(cache, layer, batch, "dr_cache_store"));
    if (!pass) return fail(DR_ERR_INVALID, "dr_cache_store: pass is NULL");
    if (pass->ctx != cache->ctx) return fail(DR_ERR_INVALID, "dr_cache_store: pass and cache use different contexts");
    if (pass->n == 0) return DR_OK;
    if (pass->max_pos >= cache->n_total)
        return fail(DR_ERR_INVALID, "dr_cache_store: position %zu >= n_total %zu", pass->max_pos,
                    cache->n_total);
    if (!k || !v) return fail(DR_ERR_INVALID, "dr_cache_store: k/v is NULL");
    DR_CHECK(use_device(cache->ctx));
    dr::StoreArgs a{};
    a.k = k;
    a.v = v;
    a.pos = pass->d_pos;
    a.pos0 = pass->max_pos - pass->min_pos + 1 == pass->n ? (int)pass->min_pos : -1;
    a.n = (int)pass->n;
    a.n_head_kv = cache->hkv[layer];
    a.hd = cache->hd[layer];
    a.cap = (int)cache->cap;
    a.kc = cache->k[layer * cache->n_batch + batch];
    a.vtc = cache->vt[layer * cache->n_batch + batch];
    a.klo = cache->klo[layer * cache->n_batch + batch];
    a.vlo = cache->vlo[layer * cache->n_batch + batch];
    a.kn_w = k_norm_w;
    a.kn_eps = eps;
    a.rstride = kv_stride ? (int)kv_stride : a.n_head_kv * a.hd;
    a.vec = a.hd == cache->hd_tile[layer] && (((uintptr_t)k | (uintptr_t)v) & 15) == 0 && a.rstride % 4 == 0;
    a.batch = (int)batch;
    a.n_batch = (int)cache->n_batch;
    a.kb = kb;
    a.vb = vb;
    a.v_norm = v_norm ? 1 : 0;
    a.rope = rope ? rope->d_table : nullptr;
    a.rot = rope ? (int)rope->rope_dim : 0;
    const size_t at = layer * cache->n_batch + batch;
    if (cache->sc[at]) {
        a.kc = reinterpret_cast<uint16_t*>(cache->k8[at]);
        a.vtc = reinterpret_cast<uint16_t*>(cache->v8[at]);
        a.sc = cache->sc[at];
        a.n_cu = cache->ctx->n_cu;
    }
    hipError_t e = a.sc ? dr::launch_store_fp8(cache->hd_tile[layer], a, cache->ctx->stream)
                        : dr::launch_store(cache->hd_tile[layer], a, cache->ctx->stream);
    if (e != hipSuccess) return hip_fail(e, "kv_store launch");
    return DR_OK;
}

// StepCache::gather of n positions on the device (pos0 >= 0: pos0, pos0 + 1, ...).
static int gather_rows(dr_step_cache* cache, size_t layer, size_t batch, const int* pos, size_t n, int pos0,
                       float* out_k, float* out_v) {
    const size_t at = layer * cache->n_batch + batch;
    dr::GatherArgs a{};
    a.kc = cache->k[at];
    a.vtc = cache->vt[at];
    a.klo = cache->klo[at];
    a.vlo = cache->vlo[at];
    a.pos = pos;
    a.n = (int)n;
    a.n_head_kv = cache->hkv[layer];
    a.hd = cache->hd[layer];
    a.cap = (int)cache->cap;
    a.out_k = out_k;
    a.out_v = out_v;
    a.pos0 = pos0;
    if (cache->sc[at]) {
        a.kc = reinterpret_cast<const uint16_t*>(cache->k8[at]);
        a.vtc = reinterpret_cast<const uint16_t*>(cache->v8[at]);
        a.sc = cache->sc[at];
        a.n_cu = cache->ctx->n_cu;
    }
    hipError_t e = a.sc ? dr::launch_gather_fp8(cache->hd_tile[layer], a, cache->ctx->stream)
                        : dr::launch_gather(cache->hd_tile[layer], a, cache->ctx->stream);
    if (e != hipSuccess) return hip_fail(e, "kv_gather launch");
    return DR_OK;
}

int dr_cache_gather_pass(dr_step_cache* cache, size_t layer, size_t batch, const dr_pass* pass, float* out_k,
                         float* out_v) {
    DR_CHECK(check_slot(cache, layer, batch, "dr_cache_gather_pass"));
    if (!pass) return fail(DR_ERR_INVALID, "dr_cache_gather_pass: pass is NULL");
    if (pass->ctx != cache->ctx)
        return fail(DR_ERR_INVALID, "dr_cache_gather_pass: pass and cache use different contexts");
    if (pass->n == 0) return DR_OK;
    if (pass->max_pos >= cache->n_total)
        return fail(DR_ERR_INVALID, "dr_cache_gather_pass: position %zu >= n_total %zu", pass->max_pos,
                    cache->n_total);
    if (!out_k || !out_v) return fail(DR_ERR_INVALID, "dr_cache_gather_pass: out_k/out_v is NULL");
    DR_CHECK(use_device(cache->ctx));
    return gather_rows(cache, layer, batch, pass->d_pos, pass->n,
                       pass->max_pos - pass->min_pos + 1 == pass->n ? (int)pass->min_pos : -1, out_k, out_v);
}

int dr_cache_gather(dr_step_cache* cache, size_t layer, size_t batch, const size_t* positions,
                    size_t n, float* out_k, float* out_v) {
    DR_CHECK(check_slot(cache, layer, batch, "dr_cache_gather"));
    if (n == 0) return DR_OK;
    if (!positions || !out_k || !out_v) return fail(DR_ERR_INVALID, "dr_cache_gather: NULL argument");
    std::vector<int32_t> h(n);
    for (size_t i = 0; i < n; ++i) {
        if (positions[i] >= cache->n_total)
            return fail(DR_ERR_INVALID, "dr_cache_gather: position %zu >= n_total %zu",
                        positions[i], cache->n_total);
        h[i] = (int32_t)positions[i];
    }
    dr_ctx* ctx = cache->ctx;
    DR_CHECK(use_device(ctx));
    DR_CHECK(ensure(ctx->meta, n * sizeof(int32_t)));
    DR_HIP(hipMemcpyAsync(ctx->meta.p, h.data(), n * sizeof(int32_t), hipMemcpyHostToDevice,
                          ctx->stream));
    DR_CHECK(gather_rows(cache, layer, batch, static_cast<const int*>(ctx->meta.p), n, -1, out_k, out_v));
    // the staging vector h dies here; the copy above was from pageable memory
    // and is complete when hipMemcpyAsync returns.
    return DR_OK;
}

namespace {

// Makes the device copy of a slot's split state current.
int state_to_device(dr_step_cache* c, dr_step_cache::Slot& s) {
    if (s.dev_state) return DR_OK;
    DR_CHECK(use_device(c->ctx));
    const size_t bytes = std::max(c->n_total, (size_t)1) * sizeof(int32_t);
    if (!s.d_prev) DR_HIP(dev_malloc(&s.d_prev, bytes));
    if (!s.d_lc) DR_HIP(dev_malloc(&s.d_lc, bytes));
    if (c->n_total > 0) {
        DR_HIP(hipMemcpyAsync(s.d_prev, s.prev_seq.data(), c->n_total * sizeof(int32_t),
                              hipMemcpyHostToDevice, c->ctx->stream));
        DR_HIP(hipMemcpyAsync(s.d_lc, s.last_changed.data(), c->n_total * sizeof(int32_t),
                              hipMemcpyHostToDevice, c->ctx->stream));
        DR_HIP(hipStreamSynchronize(c->ctx->stream));
    }
    s.dev_state = true;
    return DR_OK;
}

// Makes the host copy of a slot's split state current.
int state_to_host(dr_step_cache* c, dr_step_cache::Slot& s) {
    if (!s.dev_state) return DR_OK;
    DR_CHECK(use_device(c->ctx));
    if (c->n_total > 0) {
        DR_HIP(hipMemcpyAsync(s.prev_seq.data(), s.d_prev, c->n_total * sizeof(int32_t),
                              hipMemcpyDeviceToHost, c->ctx->stream));
        DR_HIP(hipMemcpyAsync(s.last_changed.data(), s.d_lc, c->n_total * sizeof(int32_t),
                              hipMemcpyDeviceToHost, c->ctx->stream));
        DR_HIP(hipStreamSynchronize(c->ctx->stream));
    }
    s.dev_state = false;
    return DR_OK;
}

}  // namespace

int dr_cache_update_seq_dev(dr_step_cache* cache, size_t batch, const int32_t* seq, size_t n) {
    if (!cache) return fail(DR_ERR_INVALID, "dr_cache_update_seq_dev: cache is NULL");
    if (batch >= cache->n_batch)
        return fail(DR_ERR_INVALID, "dr_cache_update_seq_dev: batch %zu >= %zu", batch, cache->n_batch);
    if (n != cache->n_total)
        return fail(DR_ERR_INVALID, "dr_cache_update_seq_dev: length %zu != n_total %zu", n, cache->n_total);
    if (n > 0 && !seq) return fail(DR_ERR_INVALID, "dr_cache_update_seq_dev: seq is NULL");
    auto& s = cache->slot[batch];
    DR_CHECK(state_to_device(cache, s));
    if (n > 0)
        DR_HIP(hipMemcpyAsync(s.d_prev, seq, n * sizeof(int32_t), hipMemcpyDeviceToDevice,
                              cache->ctx->stream));
    s.initialized = true;
    return DR_OK;
}

int dr_cache_split_active_dev(dr_step_cache* cache, size_t batch, const int32_t* seq,
                              const uint8_t* is_masked, size_t n, size_t step, dr_pass* active,
                              dr_pass* cached, size_t* n_active, size_t* n_cached) {
    if (!cache) return fail(DR_ERR_INVALID, "dr_cache_split_active_dev: cache is NULL");
    if (batch >= cache->n_batch)
        return fail(DR_ERR_INVALID, "dr_cache_split_active_dev: batch %zu >= %zu", batch, cache->n_batch);
    if (n > cache->n_total)
        return fail(DR_ERR_INVALID, "dr_cache_split_active_dev: length %zu > n_total %zu", n, cache->n_total);
    if (n > 0 && (!seq || !is_masked))
        return fail(DR_ERR_INVALID, "dr_cache_split_active_dev: seq / is_masked is NULL");
    if (!active || !cached || active == cached)
        return fail(DR_ERR_INVALID, "dr_cache_split_active_dev: need two distinct passes");
    if (active->ctx != cache->ctx || cached->ctx != cache->ctx)
        return fail(DR_ERR_INVALID, "dr_cache_split_active_dev: pass from another context");
    if (!n_active || !n_cached) return fail(DR_ERR_INVALID, "dr_cache_split_active_dev: NULL count");
    if (step > (size_t)std::numeric_limits<int32_t>::max() - 8)
        return fail(DR_ERR_INVALID, "dr_cache_split_active_dev: step too large");
    auto& s = cache->slot[batch];
    if (s.vicinity > (size_t)std::numeric_limits<int32_t>::max())
        return fail(DR_ERR_INVALID, "dr_cache_split_active_dev: vicinity too large");
    DR_CHECK(state_to_device(cache, s));
    DR_CHECK(reserve_pass(active, std::max(n, (size_t)1)));
    DR_CHECK(reserve_pass(cached, std::max(n, (size_t)1)));
    if (!cache->h_meta) {
        // the six results go straight to pinned host memory (no copy call
        // between the kernel and the synchronisation the caller waits on)
        DR_HIP(host_malloc(&cache->h_meta, 6 * sizeof(int32_t)));
        DR_HIP(hipHostGetDevicePointer(reinterpret_cast<void**>(&cache->h_meta_dev), cache->h_meta, 0));
    }
    dr::SplitArgs a{};
    a.seq = seq;
    a.is_masked = is_masked;
    a.prev_seq = s.d_prev;
    a.last_changed = s.d_lc;
    a.active = active->d_pos;
    a.cached = cached->d_pos;
    a.meta = cache->h_meta_dev;
    a.n = (int)n;
    a.step = (int)step;
    a.vicinity = (int)s.vicinity;
    hipStream_t st = cache->ctx->stream;
    hipError_t e = dr::launch_split_active(a, st);
    if (e != hipSuccess) return hip_fail(e, "split_active launch");
    DR_HIP(hipStreamSynchronize(st));
    const int32_t* m = cache->h_meta;
    active->n = (size_t)m[0];
    active->min_pos = m[0] > 0 ? (size_t)m[2] : 0;
    active->max_pos = m[0] > 0 ? (size_t)m[3] : 0;
    cached->n = (size_t)m[1];
    cached->min_pos = m[1] > 0 ? (size_t)m[4] : 0;
    cached->max_pos = m[1] > 0 ? (size_t)m[5] : 0;
    *n_active = active->n;
    *n_cached = cached->n;
    return DR_OK;
}

// GGML block geometry of the weight types dr_qmatmul runs: values and bytes
// per block (0: not built).
static void wtype_block(int wtype, size_t& qk, size_t& bytes) {
    qk = bytes = 0;
    switch (wtype) {
        case DR_WTYPE_Q4K: qk = 256, bytes = 144; break;
        case DR_WTYPE_Q6K: qk = 256, bytes = 210; break;
        case DR_WTYPE_Q4_0: qk = 32, bytes = 18; break;
        case DR_WTYPE_Q5_0: qk = 32, bytes = 22; break;
        case DR_WTYPE_Q8_0: qk = 32, bytes = 34; break;
        default: break;
    }
}

// sizes (none of them 0) that the kernels' index arithmetic holds
static bool qmm_size_ok(size_t qk, size_t rows, size_t cols, size_t n) {
    return rows > 0 && n > 0 && cols > 0 && cols % qk == 0 && rows <= (size_t)INT32_MAX &&
           cols <= (size_t)INT32_MAX / 2 && n <= (size_t)INT32_MAX / 2 &&
           (size_t)dr::qmm_rows_padded((int)n) * (cols / qk) * (qk == 32 ? 64 : 1) <= (size_t)INT32_MAX;
}

static int qmatmul_impl(dr_ctx* ctx, int wtype, const void* w, size_t rows, size_t cols, const float* act,
                        size_t n, float* out, const float* residual, const float* norm_w, float eps,
                        const char* who) {
    if (!ctx) return fail(DR_ERR_INVALID, "%s: ctx is NULL", who);
    size_t qk, bb;
    wtype_block(wtype, qk, bb);
    if (!qk)
        return fail(DR_ERR_UNSUPPORTED, "%s: weight type %d not built (Q4_0 = 2, Q5_0 = 6, Q8_0 = 8, Q4_K = 12, "
                    "Q6_K = 14)", who, wtype);
    if (cols == 0 || cols % qk != 0)
        return fail(DR_ERR_INVALID, "%s: cols %zu is not a positive multiple of %zu", who, cols, qk);
    if (n == 0 || rows == 0) return DR_OK;
    if (!w || !act || !out) return fail(DR_ERR_INVALID, "%s: NULL w / act / out", who);
    DR_CTX_USE(ctx, who);
    if (wtype == DR_WTYPE_Q4K && ((uintptr_t)w & 15))
        return fail(DR_ERR_INVALID, "%s: Q4_K blocks must start 16-byte aligned (16-byte loads)", who);
    if (((uintptr_t)w & 1) || ((uintptr_t)act & 15))
        return fail(DR_ERR_INVALID, "%s: weight blocks must start 2-byte aligned and act 16-byte aligned", who);
    if (!qmm_size_ok(qk, rows, cols, n))
        return fail(DR_ERR_INVALID, "%s: %zu x %zu x %zu too large", who, n, rows, cols);
    DR_CHECK(use_device(ctx));
    const size_t ws = qk == 32 ? dr::qmm0_workspace_bytes((int)n, (int)cols) : dr::qmm_workspace_bytes((int)n, (int)cols);
    // (with a post-norm, the rows before the norm follow, 256-byte aligned)
    const size_t tmp_off = round_up(ws, 256), tmp_bytes = norm_w ? n * rows * sizeof(float) : 0;
    DR_CHECK(grow(ctx->q8k, tmp_off + tmp_bytes, ctx->retired));
    dr::QmmArgs a{};
    a.wtype = wtype;
    a.w = w;
    a.rows = (int)rows;
    a.cols = (int)cols;
    a.act = act;
    a.n = (int)n;
    a.n_pad = dr::qmm_rows_padded((int)n);
    a.ws = ctx->q8k.p;
    a.out = out;
    a.residual = residual;
    a.norm_w = norm_w;
    a.norm_eps = eps;
    a.n_cu = ctx->n_cu;
    a.norm_tmp = norm_w ? reinterpret_cast<float*>(static_cast<char*>(ctx->q8k.p) + tmp_off) : nullptr;
    hipError_t e = dr::launch_qmatmul(a, ctx->stream);
    if (e != hipSuccess) return hip_fail(e, "qmatmul launch");
    return DR_OK;
}

int dr_qmatmul(dr_ctx* ctx, int wtype, const void* w, size_t rows, size_t cols, const float* act,
               size_t n, float* out, const float* residual) {
    return qmatmul_impl(ctx, wtype, w, rows, cols, act, n, out, residual, nullptr, 0.0f, "dr_qmatmul");
}

int dr_qmatmul_post_norm(dr_ctx* ctx, int wtype, const void* w, size_t rows, size_t cols, const float* act,
                         size_t n, float* out, const float* residual, const float* norm_w, float eps) {
    if (!norm_w) return fail(DR_ERR_INVALID, "dr_qmatmul_post_norm: norm_w is NULL");
    return qmatmul_impl(ctx, wtype, w, rows, cols, act, n, out, residual, norm_w, eps, "dr_qmatmul_post_norm");
}

int dr_qmatmul_expert(dr_ctx* ctx, int wtype, const void* w, size_t n_expert, size_t expert, size_t rows,
                      size_t cols, const float* act, size_t n, float* out, const float* residual) {
    if (!ctx) return fail(DR_ERR_INVALID, "dr_qmatmul_expert: ctx is NULL");
    if (expert >= n_expert)
        return fail(DR_ERR_INVALID, "dr_qmatmul_expert: expert index %zu out of range (%zu experts)", expert,
                    n_expert);
    size_t qk, bb;
    wtype_block(wtype, qk, bb);
    if (!qk)
        return fail(DR_ERR_UNSUPPORTED, "dr_qmatmul_expert: weight type %d not built (Q4_0 = 2, Q5_0 = 6, "
                    "Q8_0 = 8, Q4_K = 12, Q6_K = 14)", wtype);
    if (cols == 0 || cols % qk != 0)
        return fail(DR_ERR_INVALID, "dr_qmatmul_expert: cols %zu is not a positive multiple of %zu", cols, qk);
    if (!w) return fail(DR_ERR_INVALID, "dr_qmatmul_expert: w is NULL");
    const size_t expert_bytes = rows * (cols / qk) * bb;
    return qmatmul_impl(ctx, wtype, static_cast<const uint8_t*>(w) + expert * expert_bytes, rows, cols, act, n, out,
                        residual, nullptr, 0.0f, "dr_qmatmul_expert");
}

int dr_quantize_q8_0(dr_ctx* ctx, const float* act, size_t n, size_t cols, void* out) {
    if (!ctx) return fail(DR_ERR_INVALID, "dr_quantize_q8_0: ctx is NULL");
    if (cols == 0 || cols % 32 != 0)
        return fail(DR_ERR_INVALID, "dr_quantize_q8_0: cols %zu is not a positive multiple of 32", cols);
    if (n == 0) return DR_OK;
    if (!act || !out) return fail(DR_ERR_INVALID, "dr_quantize_q8_0: NULL act / out");
    if (((uintptr_t)out & 1) || ((uintptr_t)act & 15))
        return fail(DR_ERR_INVALID, "dr_quantize_q8_0: out must be 2-byte and act 16-byte aligned");
    if (cols > (size_t)INT32_MAX || (n + 31) / 32 * (cols / 32) > (size_t)INT32_MAX / 4)
        return fail(DR_ERR_INVALID, "dr_quantize_q8_0: %zu x %zu too large", n, cols);
    DR_CHECK(use_device(ctx));
    hipError_t e = dr::launch_quantize_q80(act, (int)n, (int)cols, out, ctx->stream);
    if (e != hipSuccess) return hip_fail(e, "quantize_q8_0 launch");
    return DR_OK;
}

int dr_quantize_q8k(dr_ctx* ctx, const float* act, size_t n, size_t cols, void* out) {
    if (!ctx) return fail(DR_ERR_INVALID, "dr_quantize_q8k: ctx is NULL");
    if (cols == 0 || cols % 256 != 0)
        return fail(DR_ERR_INVALID, "dr_quantize_q8k: cols %zu is not a positive multiple of 256", cols);
    if (n == 0) return DR_OK;
    if (!act || !out) return fail(DR_ERR_INVALID, "dr_quantize_q8k: NULL act / out");
    if ((uintptr_t)out & 3) return fail(DR_ERR_INVALID, "dr_quantize_q8k: out must be 4-byte aligned");
    if (cols > (size_t)INT32_MAX || n * (cols / 256) > (size_t)INT32_MAX)
        return fail(DR_ERR_INVALID, "dr_quantize_q8k: %zu x %zu too large", n, cols);
    DR_CHECK(use_device(ctx));
    hipError_t e = dr::launch_quantize_q8k(act, (int)n, (int)cols, static_cast<dr::Q8KBlock*>(out), ctx->stream);
    if (e != hipSuccess) return hip_fail(e, "quantize_q8k launch");
    return DR_OK;
}

int dr_cache_update_seq(dr_step_cache* cache, size_t batch, const int32_t* seq, size_t n) {
    if (!cache) return fail(DR_ERR_INVALID, "dr_cache_update_seq: cache is NULL");
    if (batch >= cache->n_batch) return fail(DR_ERR_INVALID, "dr_cache_update_seq: batch %zu >= %zu", batch, cache->n_batch);
    if (n != cache->n_total)
        return fail(DR_ERR_INVALID, "dr_cache_update_seq: length %zu != n_total %zu", n, cache->n_total);
    if (n > 0 && !seq) return fail(DR_ERR_INVALID, "dr_cache_update_seq: seq is NULL");
    auto& s = cache->slot[batch];
    DR_CHECK(state_to_host(cache, s));
    std::copy(seq, seq + n, s.prev_seq.begin());
    s.initialized = true;
    return DR_OK;
}

int dr_split_active(const int32_t* prev_seq, int32_t* last_changed, const int32_t* seq,
                    const uint8_t* is_masked, size_t n, size_t step, size_t vicinity,
                    size_t* active, size_t* n_active, size_t* cached, size_t* n_cached) {
    if (n > 0 && (!prev_seq || !last_changed || !seq || !is_masked || !active || !cached))
        return fail(DR_ERR_INVALID, "dr_split_active: NULL array");
    if (!n_active || !n_cached) return fail(DR_ERR_INVALID, "dr_split_active: NULL count");
    if (step > (size_t)std::numeric_limits<int32_t>::max())
        return fail(DR_ERR_INVALID, "dr_split_active: step too large");
    const int32_t st = (int32_t)step;
    // cache.rs:88-97: changed, still masked, or changed within
    // EXTRA_ACTIVE_STEPS (= 2, cache.rs:23) steps.
    std::vector<uint8_t> act(n, 0);
    for (size_t i = 0; i < n; ++i) {
        const bool changed = seq[i] != prev_seq[i];
        if (changed) last_changed[i] = st;
        const bool recent = last_changed[i] >= 0 && (st - last_changed[i]) <= 2;
        act[i] = changed || is_masked[i] || recent;
    }
    // cache.rs:98-104: vicinity refresh around still-masked positions.
    if (vicinity > 0) {
        for (size_t m = 0; m < n; ++m) {
            if (!is_masked[m]) continue;
            const size_t lo = m > vicinity ? m - vicinity : 0;
            const size_t hi = std::min(m + vicinity + 1, n);
            std::fill(act.begin() + lo, act.begin() + hi, 1);
        }
    }
    size_t na = 0, nc = 0;
    for (size_t i = 0; i < n; ++i) {
        if (act[i])
            active[na++] = i;
        else
            cached[nc++] = i;
    }
    *n_active = na;
    *n_cached = nc;
    return DR_OK;
}

int dr_cache_split_active(dr_step_cache* cache, size_t batch, const int32_t* seq,
                          const uint8_t* is_masked, size_t n, size_t step, size_t* active,
                          size_t* n_active, size_t* cached, size_t* n_cached) {
    if (!cache) return fail(DR_ERR_INVALID, "dr_cache_split_active: cache is NULL");
    if (batch >= cache->n_batch) return fail(DR_ERR_INVALID, "dr_cache_split_active: batch %zu >= %zu", batch, cache->n_batch);
    if (n > cache->n_total)
        return fail(DR_ERR_INVALID, "dr_cache_split_active: length %zu > n_total %zu", n, cache->n_total);
    auto& s = cache->slot[batch];
    DR_CHECK(state_to_host(cache, s));
    return dr_split_active(s.prev_seq.data(), s.last_changed.data(), seq, is_masked, n, step,
                           s.vicinity, active, n_active, cached, n_cached);
}

int dr_cache_set_vicinity(dr_step_cache* cache, size_t batch, size_t vicinity) {
    if (!cache || batch >= cache->n_batch) return fail(DR_ERR_INVALID, "dr_cache_set_vicinity: bad cache/batch");
    cache->slot[batch].vicinity = vicinity;
    return DR_OK;
}

int dr_cache_initialized(const dr_step_cache* cache, size_t batch) {
    if (!cache || batch >= cache->n_batch) return 0;
    return cache->slot[batch].initialized ? 1 : 0;
}

// ---------------------------------------------------------------- attention

// The plan of a hi/lo kernel, 16-row or 32-row waves: 64 query rows per
// workgroup (32-row waves at head dim 256: 128), the keys split across
// workgroups when there are too few of them to fill the chip.  tiles: key
// tiles that its busiest CU multiplies.
static dr::LaunchPlan plan_hilo_rows(dr_ctx* ctx, const dr::AttnArgs& a, int hd_tile, int max_nq, int max_nk,
                                     int mask, bool w32, int& tiles) {
    dr::LaunchPlan p{};
    p.hd_tile = hd_tile;
    p.block_n = 32;
    const int rows = w32 ? dr::hilo32_rows(hd_tile) : dr::hilo_rows();
    p.rb = rows / 32;
    p.kq = 1;
    p.waves = !w32 && hd_tile > 256 ? 8 : 4;
    p.stages = 1;
    p.rowgroups = (a.group * max_nq + rows - 1) / rows;
    p.mask = mask;
    p.w16 = !w32;
    p.kernel = dr::KERNEL_HILO;
    const int base = a.n_batch * a.n_head_kv * p.rowgroups;
    const int ntiles = std::max(1, (max_nk + 31) / 32);
    // Workgroups that run at once: the 16-row kernel takes at most 64 KB of
    // LDS up to head dim 256, so two share a CU and key splits fill both; the
    // others take a CU each.
    const int slots = ctx->n_cu * (w32 || hd_tile > 256 ? 1 : 2);
    int split = 1;
    if (ctx->force_split > 0)
        split = ctx->force_split;
    else if (2 * base <= slots)
        split = std::min(slots / std::max(base, 1), ntiles);
    p.n_split = std::max(1, split);
    p.n_workgroups = base * p.n_split;
    // a workgroup's key range: all keys, or the window around its rows
    int range = ntiles;
    if (mask == dr::MASK_POS && a.window >= 0) {
        const long long near = 2LL * a.window + std::min(max_nq, rows);
        range = (int)std::min<long long>((a.key_band + 31) / 32, (std::min<long long>(max_nk, near) + 31) / 32 + 1);
    }
    tiles = (p.n_workgroups + slots - 1) / slots * ((range + p.n_split - 1) / p.n_split);
    return p;
}

// 32-row waves (attn_hilo32_kernel) at the head dims and masks they are built
// for, or the 16-row kernel.  A 32-row tile costs less, a 32-row workgroup
// starts 2-4 us later and holds the CU alone.
// - A bias or a full rotary: 32 rows.  They are applied as Q is loaded; the
//   16-row kernel needs a copy of Q and an epilogue pass first (QK-norm and
//   RoPE, 16 / 32 rows, us with the store: 16/8 heads of 256, window 1024, 1
//   row of 65 keys 25 / 21, 64 of 576 41 / 36, 256 of 4352 56 / 46; 16/2 of
//   512 30 / 22, 53 / 42, 155 / 126).
// - Else 32 rows where the busiest CU has at least 4 key tiles (shorter
//   loops do not make up for the later start: 16/8 of 256, 1 row of 65 keys
//   12 / 15, 64 of 576 25 / 27, 256 of 320 32 / 36, 256 of 4352 66 / 61; 16/2
//   of 512, 32 of 96 19 / 19, 256 of 4352 126 / 112), where its workgroups
//   are filled to more than half (8/8 of 256, batch of 4, 2 of 1321 27 / 32;
//   16/8 of 512, batch of 2, 3 of 4173 58 / 65) and where its larger
//   workgroups leave no CU with much more to do (16/8 of 256, 659 of 7824,
//   123 tiles against 82: 225 / 242);
// - and where the 16-row kernel's second workgroup per CU would leave 48 or
//   more further splits to merge (8/4 of 256, window 512, 32 of 4128, 128
//   splits against 64: 36 / 27).
// (1580 calls without a bias or a rotary, 1-1024 rows, 32-8192 keys, windows
// and causal prefixes, batches of 1-4: 6 take more than 2 % longer than on the
// 16-row kernel, 4.7 % at most.)
static size_t hilo_q_bytes(const dr::AttnArgs& a, const dr::LaunchPlan& p);
static dr::LaunchPlan plan_hilo(dr_ctx* ctx, const dr::AttnArgs& a, int hd, int max_nq, int max_nk,
                                int mask) {
    const int hd_tile = hd_tile_for((size_t)hd);
    int l16 = 0, l32 = 0;
    const dr::LaunchPlan p16 = plan_hilo_rows(ctx, a, hd_tile, max_nq, max_nk, mask, false, l16);
    if (dr::hilo32_rows(hd_tile) == 0 || hd != hd_tile || mask == dr::MASK_KEYS) return p16;
    const dr::LaunchPlan p32 = plan_hilo_rows(ctx, a, hd_tile, max_nq, max_nk, mask, true, l32);
    if (hilo_q_bytes(a, p16) > 0 && hilo_q_bytes(a, p32) == 0) return p32;
    const bool long_loop = l32 >= 4 && 2 * a.group * max_nq >= dr::hilo32_rows(hd_tile) && 20 * l32 <= 27 * l16;
    // (forced splits: the larger row groups' partials must not outgrow the
    // fixed scratch of dr_attention_cached_noalloc)
    const bool fits = dr::split_workspace_bytes(p32, a.n_batch, a.n_head_kv) <= dr::scratch_bytes();
    return fits && (long_loop || p16.n_split - p32.n_split >= 48) ? p32 : p16;
}

static dr::LaunchPlan plan_for(dr_ctx* ctx, const dr::AttnArgs& a, int hd, int max_nq,
                               int max_nk, int mask, int qepi) {
    // a layer that keeps K's lo half gets f32-accurate scores, unless another
    // kernel family is forced (then the lo half is not read)
    if (a.fp8)
        return dr::plan_fp8(hd_tile_for((size_t)hd), a.n_batch, a.n_head_kv, a.group, max_nq, a.key_band, mask,
                            ctx->n_cu, ctx->force_split, ctx->force_rows, (int)TICKETS);
    // (the 8 bit family forced is no choice for a layer that is not 8 bit: automatic)
    const bool hilo_asked = ctx->force_kernel == dr::KERNEL_AUTO || ctx->force_kernel == dr::KERNEL_HILO ||
                            ctx->force_kernel == dr::KERNEL_FP8;
    const bool bf16_rows = a.q_bf16 || a.o_bf16;
    if (a.slot[0].klo && hilo_asked && !bf16_rows) return plan_hilo(ctx, a, hd, max_nq, max_nk, mask);
    // bf16 Q or output rows: only the per-wave-stream kernel reads / writes them
    const int kernel = bf16_rows ? dr::KERNEL_STREAMS
                                : (ctx->force_kernel >= dr::KERNEL_HILO ? dr::KERNEL_AUTO : ctx->force_kernel);
    return dr::plan_attention(hd, a.n_batch, a.n_head_kv, a.group, max_nq, max_nk, mask, qepi,
                              mask == dr::MASK_POS ? a.window : -1, a.rope ? a.rot : 0, ctx->n_cu,
                              ctx->force_rb, ctx->force_kq, ctx->force_split, ctx->force_rows, kernel,
                              ctx->merge_in_kernel != 0, a.key_band);
}

// The 16-row hi/lo kernel reads plain Q: with a Q epilogue (bias, QK-norm,
// RoPE), each batch slot's Q is copied into a workspace and the epilogue
// (qkv_epilogue.hip, Q heads only) runs there first.  Bytes of that
// workspace (0: the kernel reads the caller's rows): the QK-norm alone at a
// full head-dim tile needs none, the kernel applies it as it loads Q (a
// row's sum of squares over four lanes of one wave, or of the row block's
// two waves at hd 512).  The 32-row kernel applies all three as it loads Q
// when the rotary covers the head; in front of a partial rotary it needs the
// copy too.
static size_t hilo_q_bytes(const dr::AttnArgs& a, const dr::LaunchPlan& p) {
    if (p.kernel != dr::KERNEL_HILO || (!a.qn_w && !a.qb && !a.rope)) return 0;
    if (!p.w16 && (!a.rope || a.rot == a.hd)) return 0;
    if (!a.qb && !a.rope && a.hd == p.hd_tile) return 0;
    size_t total = 0;
    for (int b = 0; b < a.n_batch; ++b) total += (size_t)a.slot[b].nq * a.n_head * a.hd;
    return total * sizeof(float);
}

// (the copy packs the rows: the epilogue pass reads [nq][n_head * hd])
static int hilo_prepare_q(dr_ctx* ctx, dr::AttnArgs& a, float* base) {
    const size_t row = (size_t)a.n_head * a.hd;
    for (int b = 0; b < a.n_batch; ++b) {
        dr::AttnSlot& s = a.slot[b];
        const size_t n = (size_t)s.nq * row;
        if (n == 0) continue;
        DR_HIP(hipMemcpy2DAsync(base, row * sizeof(float), s.q, (size_t)a.q_rstride * sizeof(float),
                                row * sizeof(float), (size_t)s.nq, hipMemcpyDeviceToDevice, ctx->stream));
        dr::EpiArgs e{};
        e.q = base;
        e.pos = s.qpos;
        e.pos0 = s.qpos0;
        e.n = s.nq;
        e.n_head = a.n_head;
        e.n_head_kv = 0;  // Q heads only
        e.hd = a.hd;
        e.bq = a.qb;
        e.qn_w = a.qn_w;
        e.eps = a.qn_eps;
        e.rope = a.rope;
        e.rot = a.rot;
        e.vec = a.hd % 4 == 0;
        hipError_t err = dr::launch_epilogue(e, ctx->stream);
        if (err != hipSuccess) return hip_fail(err, "hi/lo attention: Q epilogue launch");
        s.q = base;
        base += n;
    }
    a.qn_w = nullptr;
    a.qb = nullptr;
    a.rope = nullptr;
    a.rot = 0;
    a.q_rstride = (int)row;
    return DR_OK;
}

// Launches plan p.  The key-split partials go to the context's workspace,
// or with fixed_ws to the library's fixed device scratch (no allocation: a
// plan that needs more than it holds is an error).
// bf16 Q rows are read by the per-wave-stream kernel only.
static int check_q_dtype(const dr::AttnArgs& a, const dr::LaunchPlan& p, const char* who) {
    if ((!a.q_bf16 && !a.o_bf16) || p.kernel == dr::KERNEL_STREAMS || p.kernel == dr::KERNEL_FP8) return DR_OK;
    return fail(DR_ERR_UNSUPPORTED,
                "%s: bf16 Q / output rows (dr_ctx_set_q_dtype, dr_ctx_set_o_dtype) are read and written by the "
                "per-wave-stream kernel only: head dim 128 or 256, no per-key masks, a Q epilogue of at most "
                "bias, QK-norm and full-rotary RoPE, no forced tile shape and no hi/lo layer",
                who);
}

static int launch_plan(dr_ctx* ctx, dr::AttnArgs& a, const dr::LaunchPlan& p, bool fixed_ws = false) {
    DR_CHECK(check_q_dtype(a, p, "attention"));
    // device memory beyond the inputs and outputs: the key-split partials,
    // and the hi/lo kernel's copy of Q with its epilogue applied
    const size_t ws = dr::split_workspace_bytes(p, a.n_batch, a.n_head_kv);
    const size_t qws = hilo_q_bytes(a, p);
    float* qpre = nullptr;
    if (fixed_ws) {
        // both in the fixed scratch, Q after the partials (256-byte aligned)
        const size_t qoff = round_up(ws, 256);
        if (qoff + qws > dr::scratch_bytes())
            return fail(DR_ERR_INVALID,
                        "dr_attention_cached_noalloc: the plan (%d key splits%s) needs %zu bytes of "
                        "workspace, more than the fixed %zu",
                        p.n_split, qws ? ", hi/lo Q epilogue" : "", qoff + qws, dr::scratch_bytes());
        char* base = static_cast<char*>(dr::scratch_ptr(ctx->device));
        if (!base) return fail(DR_ERR_HIP, "the device scratch of device %d is not set up", ctx->device);
        if (ws > 0) a.part_o = reinterpret_cast<float*>(base);
        if (qws > 0) qpre = reinterpret_cast<float*>(base + qoff);
    } else {
        if (ws > 0) {
            DR_CHECK(grow(ctx->part, ws, ctx->retired));
            a.part_o = static_cast<float*>(ctx->part.p);
        }
        if (qws > 0) {
            DR_CHECK(grow(ctx->qpre, qws, ctx->retired));
            qpre = static_cast<float*>(ctx->qpre.p);
        }
    }
    if (qpre) DR_CHECK(hilo_prepare_q(ctx, a, qpre));
    // Key splits of the per-wave-stream kernel merge in-kernel when they are
    // few enough for its registers, the context's tickets cover the row
    // blocks and the partials' byte offsets fit the kernel's 32-bit buffer
    // offsets; otherwise split_merge_kernel runs.
    a.ticket = nullptr;
    if (ctx->merge_in_kernel && p.kernel == dr::KERNEL_STREAMS && p.n_split > 1 &&
        p.n_split <= dr::ring_merge_splits(p.hd_tile)) {
        const size_t blocks = (size_t)a.n_batch * a.n_head_kv * p.rowgroups;
        if (blocks <= TICKETS && ws < ((size_t)1 << 31)) a.ticket = static_cast<int*>(ctx->tick.p);
    }
    // (an 8 bit layer's kernel always merges its own, and its plan keeps to both limits)
    if (p.kernel == dr::KERNEL_FP8 && p.n_split > 1) a.ticket = static_cast<int*>(ctx->tick.p);
    hipError_t e = dr::launch_attention(p, a, ctx->stream);
    if (e != hipSuccess) return hip_fail(e, "attention launch");
    ctx->last = p;
    ctx->last.merge = p.n_split <= 1 ? 0 : (a.ticket ? 2 : 1);
    ctx->has_last = true;
    return DR_OK;
}

static int launch_planned(dr_ctx* ctx, dr::AttnArgs& a, int hd, int max_nq, int max_nk,
                          int mask, int qepi) {
    return launch_plan(ctx, a, plan_for(ctx, a, hd, max_nq, max_nk, mask, qepi));
}

static float scale_log2(float scale) { return scale * 1.4426950408889634f; }

static int opt_to_int(dr_opt_usize o) {
    if (!o.present) return -1;
    return (int)std::min(o.value, MAX_POS);
}

// The AttnArgs of a cached attention call over items (q, out, pass per
// batch slot), validated; max_nq = 0 means every pass is empty.
static int cached_args(dr_step_cache* cache, size_t layer, const dr_batch_item* items,
                       size_t n_items, size_t n_head, dr_opt_usize sliding_window,
                       dr_opt_usize causal_prefix, float scale, const float* q_norm_w,
                       float q_norm_eps, const char* who, dr::AttnArgs& a, int& max_nq) {
    DR_CHECK(check_slot(cache, layer, 0, who));
    if (!items || n_items < 1) return fail(DR_ERR_INVALID, "%s: no items", who);
    if (n_items > cache->n_batch)
        return fail(DR_ERR_INVALID, "%s: %zu items > cache n_batch %zu", who, n_items,
                    cache->n_batch);
    const size_t hkv = (size_t)cache->hkv[layer];
    const size_t hd = (size_t)cache->hd[layer];
    if (n_head < hkv || n_head % hkv != 0)
        return fail(DR_ERR_INVALID, "n_head %zu is not a multiple of n_head_kv %zu", n_head, hkv);
    dr_ctx* ctx = cache->ctx;
    a = dr::AttnArgs{};
    a.n_batch = (int)n_items;
    a.n_head = (int)n_head;
    a.n_head_kv = (int)hkv;
    a.group = (int)(n_head / hkv);
    a.hd = (int)hd;
    a.cap = (int)cache->cap;
    a.q_rstride = a.o_rstride = (int)(n_head * hd);
    a.c = scale_log2(scale);
    a.window = opt_to_int(sliding_window);
    a.prefix = opt_to_int(causal_prefix);
    a.qn_w = q_norm_w;
    a.qn_eps = q_norm_eps;
    a.q_bf16 = ctx->q_bf16;
    a.o_bf16 = ctx->o_bf16;
    max_nq = 0;
    const int tile = cache->hd_tile[layer];
    // bf16 scores hold the 1e-2 bar up to about twice the usual
    // 1/sqrt(head_dim) scale; Gemma's kq_scale 1.0 (forward.rs:338-341) is
    // 11-23 times it and moves outputs by ~0.24 on a bf16 layer.  Such a call
    // needs a DR_PRECISION_HILO layer, unless the caller forced a kernel
    // family and so asked for bf16 scores.
    // An 8 bit layer's K is coarser (N(0, 1) rows: outputs off by 2e-2 at the
    // usual scale, 0.15 at the limit); only its own kernel reads it.
    const bool hilo_layer = cache->klo[layer * cache->n_batch] != nullptr;
    const bool fp8_layer = cache->sc[layer * cache->n_batch] != nullptr;
    a.fp8 = fp8_layer ? 1 : 0;
    if (fp8_layer && ctx->force_kernel != dr::KERNEL_AUTO && ctx->force_kernel != dr::KERNEL_FP8)
        return fail(DR_ERR_UNSUPPORTED, "%s: layer %zu is held at DR_PRECISION_FP8, which the forced kernel family "
                    "(dr_ctx_set_kernel) does not read", who, layer);
    const bool forced = ctx->force_kernel != dr::KERNEL_AUTO && (fp8_layer || ctx->force_kernel != dr::KERNEL_FP8);
    if (!hilo_layer && !forced &&
        std::fabs(scale) * std::sqrt((double)hd) > MAX_BF16_SCALE)
        return fail(DR_ERR_UNSUPPORTED,
                    "%s: scale %g is %.1f times 1/sqrt(head_dim %zu), %s; "
                    "keep layer %zu at DR_PRECISION_HILO (dr_cache_create_layers, dr_cache_set_precision), or force "
                    "a kernel family (dr_ctx_set_kernel) to accept them",
                    who, scale, std::fabs(scale) * std::sqrt((double)hd), hd,
                    fp8_layer ? "where 8 bit scores move outputs by 0.15 and more"
                              : "more than bf16 scores hold to the 1e-2 bar",
                    layer);
    if ((a.q_bf16 || a.o_bf16) && !fp8_layer && ((hd != 128 && hd != 256) || cache->klo[layer * cache->n_batch]))
        return fail(DR_ERR_UNSUPPORTED,
                    "%s: bf16 Q / output rows (dr_ctx_set_q_dtype, dr_ctx_set_o_dtype) need head dim 128 or "
                    "256 and a bf16 layer (head dim %zu%s)",
                    who, hd, cache->klo[layer * cache->n_batch] ? ", hi/lo layer" : "");
    for (size_t b = 0; b < n_items; ++b) {
        const dr_batch_item& it = items[b];
        if (!it.pass) return fail(DR_ERR_INVALID, "item %zu: pass is NULL", b);
        if (it.pass->ctx != ctx) return fail(DR_ERR_INVALID, "item %zu: pass from another context", b);
        if (it.pass->n > 0) {
            if (it.pass->max_pos >= cache->n_total)
                return fail(DR_ERR_INVALID, "item %zu: position %zu >= n_total %zu", b,
                            it.pass->max_pos, cache->n_total);
            if (!it.q || !it.out) return fail(DR_ERR_INVALID, "item %zu: q/out is NULL", b);
            if ((int)hd == tile && (((uintptr_t)it.q | (uintptr_t)it.out) & 15))
                return fail(DR_ERR_INVALID, "item %zu: q/out must be 16-byte aligned", b);
        }
        dr::AttnSlot& s = a.slot[b];
        s.q = it.q;
        s.out = it.out;
        s.qpos = it.pass->d_pos;
        s.k = cache->k[layer * cache->n_batch + b];
        s.vt = cache->vt[layer * cache->n_batch + b];
        s.klo = cache->klo[layer * cache->n_batch + b];
        s.vlo = cache->vlo[layer * cache->n_batch + b];
        if (fp8_layer) {
            s.k = reinterpret_cast<const uint16_t*>(cache->k8[layer * cache->n_batch + b]);
            s.vt = reinterpret_cast<const uint16_t*>(cache->v8[layer * cache->n_batch + b]);
            s.klo = reinterpret_cast<const uint16_t*>(cache->sc[layer * cache->n_batch + b]);
        }
        s.nq = (int)it.pass->n;
        s.nk = (int)cache->n_total;
        s.qpos_sorted = 1;  // dr_pass positions are strictly ascending
        const dr_pass* ps = it.pass;
        s.qpos0 = ps->n > 0 && ps->max_pos - ps->min_pos + 1 == ps->n ? (int)ps->min_pos : -1;
        max_nq = std::max(max_nq, s.nq);
    }
    // the keys any row block can see, for the planner: the union of the
    // items' sliding-window bands [min_pos - w + 1, max_pos + w) in the cache
    a.key_band = (int)cache->n_total;
    if (a.window >= 0) {
        long long lo = (long long)cache->n_total, hi = 0;
        for (size_t b = 0; b < n_items; ++b) {
            const dr_pass* ps = items[b].pass;
            if (ps->n == 0) continue;
            lo = std::min(lo, std::max(0LL, (long long)ps->min_pos - a.window + 1));
            hi = std::max(hi, std::min((long long)cache->n_total, (long long)ps->max_pos + a.window));
        }
        a.key_band = (int)std::max(0LL, hi - lo);
    }
    return DR_OK;
}

static int mask_of(dr_opt_usize sliding_window, dr_opt_usize causal_prefix) {
    return (sliding_window.present || causal_prefix.present) ? dr::MASK_POS : dr::MASK_NONE;
}

int dr_attention_cached(dr_step_cache* cache, size_t layer, const dr_batch_item* items,
                        size_t n_items, size_t n_head, dr_opt_usize sliding_window,
                        dr_opt_usize causal_prefix, float scale, const float* q_norm_w,
                        float q_norm_eps) {
    dr::AttnArgs a;
    int max_nq = 0;
    DR_CHECK(cached_args(cache, layer, items, n_items, n_head, sliding_window, causal_prefix,
                         scale, q_norm_w, q_norm_eps, "dr_attention_cached", a, max_nq));
    if (max_nq == 0) return DR_OK;
    DR_CTX_USE(cache->ctx, "dr_attention_cached");
    DR_CHECK(use_device(cache->ctx));
    return launch_planned(cache->ctx, a, a.hd, max_nq, (int)cache->n_total,
                          mask_of(sliding_window, causal_prefix),
                          q_norm_w ? dr::QEPI_NORM : dr::QEPI_NONE);
}

int dr_attention_cached_noalloc(dr_step_cache* cache, size_t layer, const dr_batch_item* items,
                                size_t n_items, size_t n_head, dr_opt_usize sliding_window,
                                dr_opt_usize causal_prefix, float scale, const float* q_norm_w,
                                float q_norm_eps) {
    dr::AttnArgs a;
    int max_nq = 0;
    DR_CHECK(cached_args(cache, layer, items, n_items, n_head, sliding_window, causal_prefix,
                         scale, q_norm_w, q_norm_eps, "dr_attention_cached_noalloc", a, max_nq));
    if (max_nq == 0) return DR_OK;
    dr_ctx* ctx = cache->ctx;
    DR_CTX_USE(ctx, "dr_attention_cached_noalloc");
    DR_CHECK(use_device(ctx));
    const dr::LaunchPlan p = plan_for(ctx, a, a.hd, max_nq, (int)cache->n_total,
                                      mask_of(sliding_window, causal_prefix),
                                      q_norm_w ? dr::QEPI_NORM : dr::QEPI_NONE);
    // calls on this GPU from different streams take turns with its scratch
    // (under graph capture the graph orders them)
    ScratchOrder& so = g_scratch_order[ctx->device];
    std::lock_guard<std::mutex> lk(so.mu);
    const bool cap = capturing(ctx->stream);
    if (!cap && so.last && so.last != ctx->stream) DR_HIP(hipStreamWaitEvent(ctx->stream, so.done, 0));
    DR_CHECK(launch_plan(ctx, a, p, true));
    if (!cap) {
        DR_HIP(hipEventRecord(so.done, ctx->stream));
        so.last = ctx->stream;
    }
    return DR_OK;
}

int dr_attention_step(dr_step_cache* cache, size_t layer, const dr_step_item* items,
                      size_t n_items, size_t n_head, dr_opt_usize sliding_window,
                      dr_opt_usize causal_prefix, float scale, const float* q_norm_w,
                      float q_norm_eps, const float* k_norm_w, float k_norm_eps) {
    if (!items || n_items < 1) return fail(DR_ERR_INVALID, "dr_attention_step: no items");
    if (n_items > (size_t)dr::MAX_BATCH)
        return fail(DR_ERR_INVALID, "dr_attention_step: %zu items > %d", n_items, dr::MAX_BATCH);
    dr_batch_item bi[dr::MAX_BATCH];
    for (size_t b = 0; b < n_items; ++b) bi[b] = dr_batch_item{items[b].q, items[b].out, items[b].pass};
    dr::AttnArgs a;
    int max_nq = 0;
    DR_CHECK(cached_args(cache, layer, bi, n_items, n_head, sliding_window, causal_prefix, scale,
                         q_norm_w, q_norm_eps, "dr_attention_step", a, max_nq));
    for (size_t b = 0; b < n_items; ++b)
        if (items[b].pass->n > 0 && (!items[b].k || !items[b].v))
            return fail(DR_ERR_INVALID, "item %zu: k/v is NULL", b);
    if (max_nq == 0) return DR_OK;
    DR_CTX_USE(cache->ctx, "dr_attention_step");
    DR_CHECK(use_device(cache->ctx));
    const int mask = mask_of(sliding_window, causal_prefix);
    const int qepi = q_norm_w ? dr::QEPI_NORM : dr::QEPI_NONE;
    const dr::LaunchPlan p = plan_for(cache->ctx, a, a.hd, max_nq, (int)cache->n_total, mask, qepi);
    DR_CHECK(check_q_dtype(a, p, "dr_attention_step"));  // (before any store)
    // StepCache::store of each item's active rows, then the attention over
    // the cache (two launches on the context's stream)
    for (size_t b = 0; b < n_items; ++b)
        DR_CHECK(dr_cache_store(cache, layer, b, items[b].pass, items[b].k, items[b].v, k_norm_w, k_norm_eps));
    return launch_plan(cache->ctx, a, p);
}

// dr_attention_step_epi and dr_attention_step_rows: the store of each item's
// rows (with the K / V part of the epilogue) and the attention (with its Q
// part); Q rows q_stride and K / V rows kv_stride elements apart (0: packed).
static int step_impl(dr_step_cache* cache, size_t layer, const dr_step_item* items, size_t n_items,
                     size_t n_head, dr_opt_usize sliding_window, dr_opt_usize causal_prefix, float scale,
                     const dr_epilogue* epi, size_t q_stride, size_t kv_stride, const char* who) {
    static const dr_epilogue none{};
    if (!epi) epi = &none;
    if (!items || n_items < 1) return fail(DR_ERR_INVALID, "%s: no items", who);
    if (n_items > (size_t)dr::MAX_BATCH)
        return fail(DR_ERR_INVALID, "%s: %zu items > %d", who, n_items, dr::MAX_BATCH);
    const dr_rope* rope = epi->rope;
    if (rope) {
        if (!cache || rope->ctx != cache->ctx)
            return fail(DR_ERR_INVALID, "%s: rope uses another context", who);
        if (rope->rope_dim % 8 != 0)
            return fail(DR_ERR_UNSUPPORTED, "rope_dim %zu is not a multiple of 8 (use dr_qkv_epilogue)",
                        rope->rope_dim);
        if (layer < cache->n_layer && rope->rope_dim > (size_t)cache->hd[layer])
            return fail(DR_ERR_INVALID, "rope_dim %zu > head_dim %d", rope->rope_dim, cache->hd[layer]);
        for (size_t b = 0; b < n_items; ++b)
            if (items[b].pass && items[b].pass->n > 0 && items[b].pass->max_pos >= rope->max_len)
                return fail(DR_ERR_INVALID, "item %zu: position %zu >= the RoPE table's %zu", b,
                            items[b].pass->max_pos, rope->max_len);
    }
    dr_batch_item bi[dr::MAX_BATCH];
    for (size_t b = 0; b < n_items; ++b) bi[b] = dr_batch_item{items[b].q, items[b].out, items[b].pass};
    dr::AttnArgs a;
    int max_nq = 0;
    DR_CHECK(cached_args(cache, layer, bi, n_items, n_head, sliding_window, causal_prefix, scale,
                         epi->q_norm_w, epi->eps, who, a, max_nq));
    DR_CTX_USE(cache->ctx, who);
    const size_t q_row = n_head * (size_t)a.hd, kv_row = (size_t)a.n_head_kv * a.hd;
    if (q_stride && (q_stride < q_row || q_stride > (size_t)INT32_MAX || q_stride % 4 != 0))
        return fail(DR_ERR_INVALID, "%s: q_stride %zu is not a multiple of 4 of at least n_head * head_dim %zu", who,
                    q_stride, q_row);
    if (kv_stride && (kv_stride < kv_row || kv_stride > (size_t)INT32_MAX))
        return fail(DR_ERR_INVALID, "%s: kv_stride %zu < n_head_kv * head_dim %zu", who, kv_stride, kv_row);
    if (q_stride) a.q_rstride = (int)q_stride;
    for (size_t b = 0; b < n_items; ++b)
        if (items[b].pass->n > 0 && (!items[b].k || !items[b].v))
            return fail(DR_ERR_INVALID, "item %zu: k/v is NULL", b);
    a.qb = epi->bq;
    a.rope = rope ? rope->d_table : nullptr;
    a.rot = rope ? (int)rope->rope_dim : 0;
    if (max_nq == 0) return DR_OK;  // (no row to store or to plan for)
    const int mask = mask_of(sliding_window, causal_prefix);
    const int qepi = (epi->bq || rope) ? dr::QEPI_FULL : (epi->q_norm_w ? dr::QEPI_NORM : dr::QEPI_NONE);
    const dr::LaunchPlan p = plan_for(cache->ctx, a, a.hd, max_nq, (int)cache->n_total, mask, qepi);
    DR_CHECK(check_q_dtype(a, p, who));  // (before any store)
    for (size_t b = 0; b < n_items; ++b)
        DR_CHECK(store_rows(cache, layer, b, items[b].pass, items[b].k, items[b].v, epi->k_norm_w,
                            epi->eps, epi->bk, epi->bv, epi->v_norm, rope, kv_stride));
    return launch_plan(cache->ctx, a, p);
}

int dr_attention_step_epi(dr_step_cache* cache, size_t layer, const dr_step_item* items,
                          size_t n_items, size_t n_head, dr_opt_usize sliding_window,
                          dr_opt_usize causal_prefix, float scale, const dr_epilogue* epi) {
    if (!epi) return fail(DR_ERR_INVALID, "dr_attention_step_epi: epi is NULL");
    return step_impl(cache, layer, items, n_items, n_head, sliding_window, causal_prefix, scale, epi, 0, 0,
                     "dr_attention_step_epi");
}

int dr_attention_step_rows(dr_step_cache* cache, size_t layer, const dr_step_item_rows* items,
                           size_t n_items, size_t n_head, dr_opt_usize sliding_window,
                           dr_opt_usize causal_prefix, float scale, const dr_epilogue* epi) {
    if (!items || n_items < 1) return fail(DR_ERR_INVALID, "dr_attention_step_rows: no items");
    if (n_items > (size_t)dr::MAX_BATCH)
        return fail(DR_ERR_INVALID, "dr_attention_step_rows: %zu items > %d", n_items, dr::MAX_BATCH);
    dr_step_item it[dr::MAX_BATCH];
    for (size_t b = 0; b < n_items; ++b) {
        if (items[b].q_stride != items[0].q_stride || items[b].kv_stride != items[0].kv_stride)
            return fail(DR_ERR_INVALID, "dr_attention_step_rows: item %zu has other strides than item 0", b);
        it[b] = dr_step_item{items[b].q, items[b].out, items[b].pass, items[b].k, items[b].v};
    }
    return step_impl(cache, layer, it, n_items, n_head, sliding_window, causal_prefix, scale, epi,
                     items[0].q_stride, items[0].kv_stride, "dr_attention_step_rows");
}

int dr_attention(float* out, size_t out_len, const float* q, size_t q_len, const float* k,
                 size_t k_len, const float* v, size_t v_len, dr_attn_shape s, dr_rows qr,
                 dr_rows kr) {
    // Contract of attention.rs:106-109 (debug_asserts) plus the slice bounds
    // the row kernels index (:143-152).
    const size_t nq = s.nq, nk = s.nk, h = s.n_head, hkv = s.n_head_kv, hd = s.head_dim;
    if (out_len != nq * h * hd)
        return fail(DR_ERR_INVALID, "out.len() %zu != nq*n_head*head_dim %zu", out_len, nq * h * hd);
    if (qr.pos_len != nq) return fail(DR_ERR_INVALID, "qr.pos.len() %zu != nq %zu", qr.pos_len, nq);
    if (kr.pos_len != nk) return fail(DR_ERR_INVALID, "kr.pos.len() %zu != nk %zu", kr.pos_len, nk);
    if (nq == 0 || h == 0 || hd == 0) return DR_OK;  // no (head, query) task writes anything
    if (hkv == 0 || h % hkv != 0)
        return fail(DR_ERR_INVALID, "n_head %zu is not a multiple of n_head_kv %zu", h, hkv);
    if (hd > 512) return fail(DR_ERR_UNSUPPORTED, "head_dim %zu > 512 not built", hd);
    if (!out || !q) return fail(DR_ERR_INVALID, "out/q is NULL");
    if (q_len < nq * h * hd) return fail(DR_ERR_INVALID, "q.len() %zu < %zu", q_len, nq * h * hd);
    if (nk > 0) {
        if (!k || !v) return fail(DR_ERR_INVALID, "k/v is NULL");
        if (k_len < nk * hkv * hd) return fail(DR_ERR_INVALID, "k.len() %zu < %zu", k_len, nk * hkv * hd);
        if (v_len < nk * hkv * hd) return fail(DR_ERR_INVALID, "v.len() %zu < %zu", v_len, nk * hkv * hd);
    }
    if ((qr.pos_len && !qr.pos) || (kr.pos_len && !kr.pos) || (qr.seq_len && !qr.seq) ||
        (kr.seq_len && !kr.seq) || (qr.prefix_len && !qr.prefix))
        return fail(DR_ERR_INVALID, "row metadata pointer is NULL with nonzero length");
    if (qr.prefix_len != 0 && qr.prefix_len < nq)
        return fail(DR_ERR_INVALID, "qr.prefix.len() %zu < nq %zu", qr.prefix_len, nq);

    // Row metadata as int32 (positions and ids must fit).
    const bool masked = s.sliding_window.present || s.causal_prefix.present || qr.prefix_len > 0 ||
                        qr.seq_len > 0 || kr.seq_len > 0;
    bool kident = true;
    for (size_t j = 0; j < nk; ++j) {
        if (kr.pos[j] >= MAX_POS) return fail(DR_ERR_INVALID, "kr.pos[%zu] too large", j);
        kident = kident && kr.pos[j] == j;
    }
    for (size_t i = 0; i < nq; ++i)
        if (qr.pos[i] >= MAX_POS) return fail(DR_ERR_INVALID, "qr.pos[%zu] too large", i);
    auto seq_ok = [](const dr_rows& r) {
        for (size_t i = 0; i < r.seq_len; ++i)
            if (r.seq[i] >= MAX_POS) return false;
        return true;
    };
    if (!seq_ok(qr) || !seq_ok(kr)) return fail(DR_ERR_INVALID, "sequence id too large");
    // Layout of the int32 metadata block: qpos | qseq | qprefix | kpos | kseq
    const bool has_qseq = qr.seq_len > 0, has_kseq = kr.seq_len > 0;
    const bool has_qpref = qr.prefix_len > 0, has_kpos = masked && !kident;
    std::vector<int32_t> meta;
    meta.reserve(3 * nq + 2 * nk);
    size_t off_qpos = meta.size();
    for (size_t i = 0; i < nq; ++i) meta.push_back((int32_t)qr.pos[i]);
    size_t off_qseq = meta.size();
    if (has_qseq)
        for (size_t i = 0; i < nq; ++i) meta.push_back(i < qr.seq_len ? (int32_t)qr.seq[i] : 0);
    size_t off_qpref = meta.size();
    if (has_qpref)
        for (size_t i = 0; i < nq; ++i)
            meta.push_back((int32_t)std::min(qr.prefix[i], MAX_POS));
    size_t off_kpos = meta.size();
    if (has_kpos)
        for (size_t j = 0; j < nk; ++j) meta.push_back((int32_t)kr.pos[j]);
    size_t off_kseq = meta.size();
    if (has_kseq)
        for (size_t j = 0; j < nk; ++j) meta.push_back(j < kr.seq_len ? (int32_t)kr.seq[j] : 0);

    std::lock_guard<std::mutex> lock(g_default_mu);
    if (!g_default_ctx) DR_CHECK(dr_ctx_create(0, &g_default_ctx));
    dr_ctx* ctx = g_default_ctx;
    DR_CHECK(use_device(ctx));

    if (nk == 0) {  // every row sees no key: 0 * (1/0) = NaN (attention.rs:181-185)
        std::fill(out, out + out_len, std::numeric_limits<float>::quiet_NaN());
        return DR_OK;
    }

    const int tile = hd_tile_for(hd);
    const size_t cap = round_up(nk, dr::KEY_ALIGN);
    const size_t qb = nq * h * hd * sizeof(float), kvb = nk * hkv * hd * sizeof(float);
    const size_t cb = hkv * cap * tile * sizeof(uint16_t);
    DR_CHECK(ensure(ctx->q, qb));
    DR_CHECK(ensure(ctx->k, kvb));
    DR_CHECK(ensure(ctx->v, kvb));
    DR_CHECK(ensure(ctx->kc, cb));
    DR_CHECK(ensure(ctx->vtc, cb));
    DR_CHECK(ensure(ctx->kclo, cb));
    DR_CHECK(ensure(ctx->vtclo, cb));
    DR_CHECK(ensure(ctx->out, qb));
    DR_CHECK(ensure(ctx->meta, std::max(meta.size(), (size_t)1) * sizeof(int32_t)));
    hipStream_t st = ctx->stream;
    DR_HIP(hipMemcpyAsync(ctx->q.p, q, qb, hipMemcpyHostToDevice, st));
    DR_HIP(hipMemcpyAsync(ctx->k.p, k, kvb, hipMemcpyHostToDevice, st));
    DR_HIP(hipMemcpyAsync(ctx->v.p, v, kvb, hipMemcpyHostToDevice, st));
    DR_HIP(hipMemcpyAsync(ctx->meta.p, meta.data(), meta.size() * sizeof(int32_t),
                          hipMemcpyHostToDevice, st));
    DR_HIP(hipMemsetAsync(ctx->kc.p, 0, cb, st));
    DR_HIP(hipMemsetAsync(ctx->vtc.p, 0, cb, st));
    DR_HIP(hipMemsetAsync(ctx->kclo.p, 0, cb, st));
    DR_HIP(hipMemsetAsync(ctx->vtclo.p, 0, cb, st));

    // Pack K/V into the cache layout (key j at row j), with the lo halves
    // bf16(x - bf16(x)) beside them: the drop-in computes attention() on its
    // f32 inputs with the hi/lo kernel (f32-accurate scores and values), so
    // it meets the f32 reference's bar under every mask, including the
    // sparse ones where an output averages only a few V rows and bf16
    // operands alone would move it by up to ~1e-2.  The host copies dominate
    // this entry point's cost.
    dr::StoreArgs sa{};
    sa.k = static_cast<const float*>(ctx->k.p);
    sa.v = static_cast<const float*>(ctx->v.p);
    sa.pos = nullptr;
    sa.n = (int)nk;
    sa.n_head_kv = (int)hkv;
    sa.hd = (int)hd;
    sa.cap = (int)cap;
    sa.kc = static_cast<uint16_t*>(ctx->kc.p);
    sa.vtc = static_cast<uint16_t*>(ctx->vtc.p);
    sa.klo = static_cast<uint16_t*>(ctx->kclo.p);
    sa.vlo = static_cast<uint16_t*>(ctx->vtclo.p);
    sa.vec = (int)hd == tile;
    hipError_t e = dr::launch_store(tile, sa, st);
    if (e != hipSuccess) return hip_fail(e, "pack launch");

    const int32_t* m = static_cast<const int32_t*>(ctx->meta.p);
    dr::AttnArgs a{};
    a.n_batch = 1;
    a.n_head = (int)h;
    a.n_head_kv = (int)hkv;
    a.group = (int)(h / hkv);
    a.hd = (int)hd;
    a.cap = (int)cap;
    a.q_rstride = a.o_rstride = (int)(h * hd);
    a.c = scale_log2(s.scale);
    a.window = opt_to_int(s.sliding_window);
    a.prefix = opt_to_int(s.causal_prefix);
    dr::AttnSlot& sl = a.slot[0];
    sl.q = ctx->q.p;
    sl.out = static_cast<float*>(ctx->out.p);
    sl.qpos = m + off_qpos;
    sl.qseq = has_qseq ? m + off_qseq : nullptr;
    sl.qprefix = has_qpref ? m + off_qpref : nullptr;
    sl.k = static_cast<const uint16_t*>(ctx->kc.p);
    sl.vt = static_cast<const uint16_t*>(ctx->vtc.p);
    sl.klo = static_cast<const uint16_t*>(ctx->kclo.p);
    sl.vlo = static_cast<const uint16_t*>(ctx->vtclo.p);
    sl.kpos = has_kpos ? m + off_kpos : nullptr;
    sl.kseq = has_kseq ? m + off_kseq : nullptr;
    sl.nq = (int)nq;
    sl.nk = (int)nk;
    bool sorted = true;
    for (size_t i = 1; i < nq && sorted; ++i) sorted = qr.pos[i] > qr.pos[i - 1];
    sl.qpos_sorted = sorted ? 1 : 0;
    sl.qpos0 = -1;  // the drop-in reads each row's position
    const int mask = !masked ? dr::MASK_NONE
                             : ((has_kpos || has_kseq) ? dr::MASK_KEYS : dr::MASK_POS);
    DR_CHECK(launch_planned(ctx, a, (int)hd, (int)nq, (int)nk, mask, dr::QEPI_NONE));
    DR_HIP(hipMemcpyAsync(out, ctx->out.p, qb, hipMemcpyDeviceToHost, st));
    DR_HIP(hipStreamSynchronize(st));
    return DR_OK;
}

long dr_debug_alloc_count(void) { return g_allocs.load(std::memory_order_relaxed); }

int dr_debug_qmm_plan(int wtype, size_t rows, size_t cols, size_t n, int n_cu, int* slices, size_t* max_offset,
                      size_t* workgroups) {
    size_t qk, bb;
    wtype_block(wtype, qk, bb);
    if (!qk) return fail(DR_ERR_UNSUPPORTED, "dr_debug_qmm_plan: weight type %d not built", wtype);
    if (!slices || !max_offset || !workgroups || !qmm_size_ok(qk, rows, cols, n))
        return fail(DR_ERR_INVALID, "dr_debug_qmm_plan: %zu x %zu x %zu", n, rows, cols);
    const bool sl = dr::qmm_slices(wtype, (int)rows, (int)cols, (int)n, n_cu);
    *slices = sl ? 1 : 0;
    *max_offset = sl ? dr::qmm_slice_offset(wtype, (int)cols, (int)n) : 0;
    *workgroups = sl ? dr::qmm_slice_workgroups((int)rows, (int)n)
                     : (rows + 31) / 32 * ((size_t)dr::qmm_rows_padded((int)n) / 128);
    return DR_OK;
}

int dr_debug_ring_tiles(size_t head_dim, size_t nk, size_t cap, long long window, long long qmin,
                        long long qmax, size_t n_split, int* min_tile, int* max_tile, int* partition_ok) {
    if (dr::ring_waves((int)head_dim, 1) == 0)
        return fail(DR_ERR_UNSUPPORTED, "no stream kernel at head_dim %zu", head_dim);
    if (!min_tile || !max_tile || !partition_ok || n_split < 1 || nk > cap || cap % dr::KEY_ALIGN != 0 ||
        cap == 0 || cap >= MAX_POS)
        return fail(DR_ERR_INVALID, "dr_debug_ring_tiles: bad arguments");
    // the workgroup's key tile range, as the kernel derives it
    int kt_lo = 0, kt_hi = (int)((nk + 31) / 32);
    if (window >= 0) {
        if (window >= (long long)MAX_POS || qmin < 0 || qmax < qmin || qmax >= (long long)MAX_POS)
            return fail(DR_ERR_INVALID, "dr_debug_ring_tiles: bad window or query range");
        dr::band_tile_range((int)nk, (int)window, (int)qmin, (int)qmax, kt_lo, kt_hi);
    }
    const int cap_tiles = (int)(cap / 32);
    int lo = INT32_MAX, hi = INT32_MIN;
    bool ok = true;
    std::vector<int> mult(cap_tiles, 0);
    for (int split = 0; split < (int)n_split; ++split) {
        int t0, t1;
        dr::split_tile_range(kt_lo, kt_hi, (int)n_split, split, t0, t1);
        for (int rg = 0; rg < 24; ++rg) {  // (a rotated walk only reorders each wave's tiles)
          for (int rw = 4; rw <= 8; rw += 4) {  // every wave count built
            if (!dr::ring_waves_built((int)head_dim, rw)) continue;
            std::vector<int> seen(cap_tiles, 0);
            for (int w = 0; w < rw; ++w) {
                const dr::RingWaveTiles wt(t0, t1 - t0, w, rw, rg, cap_tiles);
                const int f = wt.first_dma();
                lo = std::min(lo, f);
                hi = std::max(hi, f);
                for (int k = 0; k < wt.kw; ++k) {
                    const int t = wt.at(k);
                    lo = std::min(lo, t);
                    hi = std::max(hi, t);
                    if (t < t0 || t >= t1 || t < 0 || t >= cap_tiles) {
                        ok = false;
                    } else {
                        ++seen[t];
                    }
                }
            }
            for (int t = 0; t < cap_tiles; ++t) {
                const bool in = t >= t0 && t < t1;
                if (seen[t] != (in ? 1 : 0)) ok = false;
                if (rg == 0 && rw == 4) mult[t] += seen[t];
            }
          }
        }
    }
    // the splits together cover the range once
    for (int t = 0; t < cap_tiles; ++t)
        if (mult[t] != ((t >= kt_lo && t < kt_hi) ? 1 : 0)) ok = false;
    *min_tile = lo;
    *max_tile = hi;
    *partition_ok = ok ? 1 : 0;
    return DR_OK;
}

}  // extern "C"
