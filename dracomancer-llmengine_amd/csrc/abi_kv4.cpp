// abi_kv4.cpp -- the paged 4-bit KV cache: argument checks of the entry points
// declared in include/draco_hip.h and their launches (kv_plan.hip, kv4.hip,
// kv4_attn.hip).
//
// No reference counterpart: the reference's caches are fp32 host arrays of one
// sequence (src/m6_engine.c:396-406).  Device pointers, enqueued on the
// caller's stream and not waited for; nothing is allocated, so every call can
// be captured.
#include <math.h>

#include "../../include/draco_hip.h"
#include "kv4.h"
#include "runtime.h"

using namespace draco;

namespace {

constexpr int MAX_DEVICES = 64;

// The stream's device made current for a call (the library's stream and
// device for NULL), the caller's restored after it.
class OnDevice {
  public:
    int enter(void* stream, hipStream_t* st) {
        if (int rc = hip(hipGetDevice(&before_), "hipGetDevice")) return rc;
        now_ = before_;
        if (!stream) {
            if (int rc = ensure_init()) return rc;  // makes the library's device current on first use
            *st = draco::stream();
        } else {
            *st = (hipStream_t)stream;
        }
        if (int rc = hip(hipStreamGetDevice(*st, &now_), "hipStreamGetDevice")) return rc;
        int cur = -1;
        if (int rc = hip(hipGetDevice(&cur), "hipGetDevice")) return rc;
        return cur == now_ ? 0 : hip(hipSetDevice(now_), "hipSetDevice");
    }
    int device() const { return now_; }
    ~OnDevice() {
        int cur = before_;
        if (before_ >= 0 && hipGetDevice(&cur) == hipSuccess && cur != before_) (void)hipSetDevice(before_);
    }

  private:
    static int hip(hipError_t e, const char* what) {
        return e == hipSuccess ? 0 : fail(-2, "kv4: %s failed: %s", what, hipGetErrorString(e));
    }
    int before_ = -1, now_ = -1;
};

int cus_of(int device) {
    static int n[MAX_DEVICES] = {};
    if (device < 0 || device >= MAX_DEVICES) return 256;
    if (!n[device]) {
        int v = 0;
        if (hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || v < 1) v = 256;
        if (v > KV4_MAX_BLOCKS / 2) v = KV4_MAX_BLOCKS / 2;
        n[device] = v;
    }
    return n[device];
}

// Slots are ints, and a step of keys behind the last slot still is one.
constexpr long MAX_SLOTS = 0x7FFFFF00L;
bool page_size_ok(int ps) { return ps >= 16 && ps <= 256 && (ps & (ps - 1)) == 0; }
bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

int view_of(const DracoKv4* c, Kv4View* v, const char* who) {
    if (!c || !c->data) return fail(-1, "%s: no cache", who);
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return fail(-1, "%s: head dim %d not in {64, 128, 256}", who, c->head_dim);
    if (!page_size_ok(c->page_size)) return fail(-1, "%s: page size %d is no power of two in 16 .. 256", who, c->page_size);
    if (c->n_kv < 1 || c->n_kv > 4096 || c->n_pages < 1 || (long)c->n_pages * c->page_size > MAX_SLOTS)
        return fail(-1, "%s: bad cache: %d KV heads, %d pages of %d", who, c->n_kv, c->n_pages, c->page_size);
    if (!aligned(c->data, 16)) return fail(-1, "%s: the pages are not 16-byte aligned", who);
    v->data = (uint8_t*)c->data;
    v->head_bytes = (int)kv4_head_bytes(c->page_size, c->head_dim);
    v->page_bytes = (unsigned)v->head_bytes * (unsigned)c->n_kv;
    v->n_pages = c->n_pages;
    v->ps_shift = __builtin_ctz((unsigned)c->page_size);
    v->n_kv = c->n_kv;
    v->hd = c->head_dim;
    return 0;
}

int type_of(int code, bool* f16, const char* who) {
    if (code != DRACO_F16 && code != DRACO_F32) return fail(-1, "%s: type code %d is neither F16 (7) nor F32 (9)", who, code);
    *f16 = code == DRACO_F16;
    return 0;
}

// Rows of n heads: 16-byte aligned, a stride of a multiple of 8 elements that
// does not overlap tokens.
int rows_ok(const void* p, long stride, long width, const char* name, const char* who) {
    if (!p) return fail(-1, "%s: %s is null", who, name);
    if (!aligned(p, 16) || stride % 8) return fail(-1, "%s: %s rows are not 16-byte aligned", who, name);
    if (stride < width) return fail(-1, "%s: %s stride %ld is less than a token's %ld values", who, name, stride, width);
    return 0;
}

int heads_ok(int n_head, int n_kv, const char* who) {
    if (n_head < 1 || n_head % n_kv || n_head > 4096) return fail(-1, "%s: %d q heads over %d KV heads", who, n_head, n_kv);
    return 0;
}

int batch_ok(int n_seq, int max_blocks, int n_pages, int page_size, const char* who) {
    if (n_seq < 0 || max_blocks < 1 || n_pages < 1) return fail(-1, "%s: bad batch: %d sequences, %d blocks, %d pages", who, n_seq, max_blocks, n_pages);
    if (!page_size_ok(page_size)) return fail(-1, "%s: page size %d is no power of two in 16 .. 256", who, page_size);
    if ((long)n_pages * page_size > MAX_SLOTS || (long)max_blocks * page_size > MAX_SLOTS)
        return fail(-1, "%s: more than 2^31 - 256 slots", who);
    return 0;
}

int too_large(const char* who) { return fail(-1, "%s: the batch needs more blocks than a launch has", who); }
int launched(int rc, const char* who) {
    if (rc) return too_large(who);
    DRACO_HIP(hipGetLastError());
    return 0;
}

int attn_args(const DracoKv4* cache, const DracoKv4Attn* p, Kv4AttnArgs* a, bool* f16) {
    const char* who = "draco_kv4_attn";
    if (!p) return fail(-1, "%s: no arguments", who);
    if (int rc = view_of(cache, &a->c, who)) return rc;
    if (int rc = type_of(p->code, f16, who)) return rc;
    if (int rc = heads_ok(p->n_head, cache->n_kv, who)) return rc;
    if (int rc = batch_ok(p->n_seq, p->max_blocks, cache->n_pages, cache->page_size, who)) return rc;
    if (p->n_tok < 0 || (long)p->n_tok * p->n_head > MAX_SLOTS) return fail(-1, "%s: n_tok %d", who, p->n_tok);
    if (p->n_tok > 0 && p->n_seq > 0 && (p->max_q < 1 || p->max_len < 0))
        return fail(-1, "%s: max_q %d, max_len %d", who, p->max_q, p->max_len);
    if (p->window < 0 || p->sink < 0) return fail(-1, "%s: window %d, sink %d", who, p->window, p->sink);
    if (!(p->scale >= 1e-12f && p->scale <= 1e12f)) return fail(-1, "%s: scale %g", who, p->scale);
    return 0;
}

Kv4AttnPlan plan_of(const DracoKv4* c, const DracoKv4Attn* p, bool f16, int cus) {
    const int max_q = p->max_q < p->n_tok ? p->max_q : p->n_tok;
    long keys = p->max_len;  // that a row sees, at most
    if (p->window > 0 && (long)p->window + p->sink < keys) keys = (long)p->window + p->sink;
    return kv4_attn_plan(c->head_dim, f16, p->n_seq, p->n_tok, p->n_head, c->n_kv, max_q, keys, cus);
}

}  // namespace

extern "C" {

size_t draco_kv4_page_bytes(int page_size, int n_kv, int head_dim) {
    if (!page_size_ok(page_size) || n_kv < 1 || (head_dim != 64 && head_dim != 128 && head_dim != 256)) return 0;
    return kv4_head_bytes(page_size, head_dim) * (size_t)n_kv;
}

int draco_kv_plan(const DracoKvPlan* p, void* stream) {
    std::lock_guard<std::recursive_mutex> g(api_mutex());
    const char* who = "draco_kv_plan";
    if (!p) return fail(-1, "%s: no arguments", who);
    if (int rc = batch_ok(p->n_seq, p->max_blocks, p->n_pages, p->page_size, who)) return rc;
    if (p->n_tok < 0 || p->n_tok > 1 << 30) return fail(-1, "%s: n_tok %d", who, p->n_tok);
    if ((p->n_seq > 0 && (!p->block_table || !p->kv_len || !p->q_len || !p->kv_len_out)) || !p->free_list || !p->n_free ||
        !p->cu_q || (p->n_tok > 0 && !p->slot) || !p->n_free_out || !p->status || !p->work)
        return fail(-1, "%s: null pointer", who);
    OnDevice dev;
    hipStream_t st;
    if (int rc = dev.enter(stream, &st)) return rc;
    const KvPlanArgs a = {p->n_seq, p->max_blocks, p->n_pages, __builtin_ctz((unsigned)p->page_size), p->n_tok,
                          p->block_table, p->kv_len, p->q_len, p->free_list, p->n_free,
                          p->cu_q, p->pos, p->slot, p->kv_len_out, p->n_free_out, p->status, p->work};
    return launched(kv_plan(a, st), who);
}

int draco_kv_release(const DracoKvRelease* p, void* stream) {
    std::lock_guard<std::recursive_mutex> g(api_mutex());
    const char* who = "draco_kv_release";
    if (!p) return fail(-1, "%s: no arguments", who);
    if (int rc = batch_ok(p->n_seq, p->max_blocks, p->n_pages, p->page_size, who)) return rc;
    if ((p->n_seq > 0 && (!p->block_table || !p->block_table_out || !p->kv_len || !p->keep || !p->kv_len_out)) ||
        !p->free_list || !p->n_free || !p->n_free_out || !p->work)
        return fail(-1, "%s: null pointer", who);
    OnDevice dev;
    hipStream_t st;
    if (int rc = dev.enter(stream, &st)) return rc;
    const KvReleaseArgs a = {p->n_seq, p->max_blocks, p->n_pages, __builtin_ctz((unsigned)p->page_size), p->block_table,
                             p->block_table_out, p->kv_len, p->keep, p->free_list, p->n_free, p->kv_len_out, p->n_free_out,
                             p->work};
    return launched(kv_release(a, st), who);
}

int draco_kv4_append(const DracoKv4* cache, const DracoKv4Append* p, void* stream) {
    std::lock_guard<std::recursive_mutex> g(api_mutex());
    const char* who = "draco_kv4_append";
    if (!p) return fail(-1, "%s: no arguments", who);
    Kv4AppendArgs a = {};
    bool f16 = false;
    if (int rc = view_of(cache, &a.c, who)) return rc;
    if (int rc = type_of(p->code, &f16, who)) return rc;
    if (p->n_head != 0)
        if (int rc = heads_ok(p->n_head, cache->n_kv, who)) return rc;
    if (p->n_tok < 0) return fail(-1, "%s: n_tok %d", who, p->n_tok);
    if (p->n_tok == 0) return 0;
    const long hd = cache->head_dim;
    if (p->n_head)
        if (int rc = rows_ok(p->q, p->q_stride, p->n_head * hd, "q", who)) return rc;
    if (p->n_head)
        if (int rc = rows_ok(p->q_out, p->q_out_stride, p->n_head * hd, "q_out", who)) return rc;
    if (int rc = rows_ok(p->k, p->k_stride, cache->n_kv * hd, "k", who)) return rc;
    if (int rc = rows_ok(p->v, p->v_stride, cache->n_kv * hd, "v", who)) return rc;
    if (!p->slot) return fail(-1, "%s: slot is null", who);
    if (p->rot < 0 || p->rot > hd || p->rot % 8) return fail(-1, "%s: rot %d is no multiple of 8 up to the head dim", who, p->rot);
    if (p->rot) {
        if (!p->pos || !p->table || p->table_rows < 1) return fail(-1, "%s: rotation without positions or table", who);
        if (!aligned(p->table, 8)) return fail(-1, "%s: the rotary table is not 8-byte aligned", who);
        if (p->pairing != 0 && p->pairing != 1) return fail(-1, "%s: pairing %d", who, p->pairing);
        if (p->n_axes < 1 || p->n_axes > 4 || (p->n_axes > 1 && p->pos_stride < p->n_tok))
            return fail(-1, "%s: %d axes with positions %ld apart", who, p->n_axes, p->pos_stride);
        for (int i = 0; i < p->rot / 2; i++) {
            if (p->axis[i] >= p->n_axes) return fail(-1, "%s: pair %d is on axis %d of %d", who, i, p->axis[i], p->n_axes);
            a.axis[i / 16] |= (uint32_t)p->axis[i] << (2 * (i % 16));
        }
    }
    // q_out may be q itself (each value is written by the lane that read it
    // only where pairs are consecutive; halves read each other's)
    if (p->n_head && p->rot && p->pairing == 1 && p->q == p->q_out) return fail(-1, "%s: q_out is q with pairs in halves", who);
    // .. and where a token's row of one is its row of the other
    if (p->n_head && p->n_tok > 1 && p->q == p->q_out && p->q_stride != p->q_out_stride)
        return fail(-1, "%s: q_out is q with strides %ld and %ld", who, p->q_stride, p->q_out_stride);
    a.q = p->q;
    a.k = p->k;
    a.v = p->v;
    a.q_out = p->q_out;
    a.q_stride = p->q_stride;
    a.q_out_stride = p->q_out_stride;
    a.k_stride = p->k_stride;
    a.v_stride = p->v_stride;
    a.slot = p->slot;
    a.n_tok = p->n_tok;
    a.n_head = p->n_head;
    a.rot = p->rot;
    a.n_axes = p->n_axes;
    a.pos = p->pos;
    a.pos_stride = p->n_axes > 1 ? p->pos_stride : 0;
    a.table = p->table;
    a.table_rows = p->table_rows;
    if (kv4_append_grid(a).blocks > KV4_MAX_GRID) return too_large(who);
    OnDevice dev;
    hipStream_t st;
    if (int rc = dev.enter(stream, &st)) return rc;
    return launched(kv4_append(a, f16, p->pairing == 1, st), who);
}

int draco_kv4_read(const DracoKv4* cache, const int* slot, int n, float* k, float* v, void* stream) {
    std::lock_guard<std::recursive_mutex> g(api_mutex());
    const char* who = "draco_kv4_read";
    Kv4View c;
    if (int rc = view_of(cache, &c, who)) return rc;
    if (n < 0) return fail(-1, "%s: n %d", who, n);
    if (n == 0) return 0;
    if (!slot || !k || !v) return fail(-1, "%s: null pointer", who);
    if (!aligned(k, 16) || !aligned(v, 16)) return fail(-1, "%s: k or v is not 16-byte aligned", who);
    if (kv4_read_grid(c, n) > KV4_MAX_GRID) return too_large(who);
    OnDevice dev;
    hipStream_t st;
    if (int rc = dev.enter(stream, &st)) return rc;
    return launched(kv4_read(c, slot, n, k, v, st), who);
}

size_t draco_kv4_attn_workspace(const DracoKv4* cache, const DracoKv4Attn* p) {
    std::lock_guard<std::recursive_mutex> g(api_mutex());
    Kv4AttnArgs a = {};
    bool f16 = false;
    if (attn_args(cache, p, &a, &f16)) return 0;
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) dev = 0;
    return kv4_attn_workspace(cache->head_dim, cus_of(dev));
}

int draco_kv4_attn(const DracoKv4* cache, const DracoKv4Attn* p, void* stream) {
    std::lock_guard<std::recursive_mutex> g(api_mutex());
    const char* who = "draco_kv4_attn";
    Kv4AttnArgs a = {};
    bool f16 = false;
    if (int rc = attn_args(cache, p, &a, &f16)) return rc;
    if (p->n_tok == 0 || p->n_seq == 0) return 0;
    const long width = (long)p->n_head * cache->head_dim;
    if (int rc = rows_ok(p->q, p->q_stride, width, "q", who)) return rc;
    if (int rc = rows_ok(p->out, p->out_stride, width, "out", who)) return rc;
    if (p->out == p->q) return fail(-1, "%s: out is q", who);
    if (!p->cu_q || !p->kv_len || !p->block_table) return fail(-1, "%s: null pointer", who);
    OnDevice dev;
    hipStream_t st;
    if (int rc = dev.enter(stream, &st)) return rc;
    const Kv4AttnPlan plan = plan_of(cache, p, f16, cus_of(dev.device()));
    if (plan.work > p->work_bytes || (plan.work && !p->work))
        return fail(-1, "%s: a workspace of %zu bytes, %zu needed", who, p->work ? p->work_bytes : 0, plan.work);
    if (plan.work && !aligned(p->work, 16)) return fail(-1, "%s: the workspace is not 16-byte aligned", who);
    a.q = p->q;
    a.out = p->out;
    a.q_stride = p->q_stride;
    a.out_stride = p->out_stride;
    a.cu_q = p->cu_q;
    a.kv_len = p->kv_len;
    a.block_table = p->block_table;
    a.n_seq = p->n_seq;
    a.n_tok = p->n_tok;
    a.n_head = p->n_head;
    a.group = p->n_head / cache->n_kv;
    a.max_blocks = p->max_blocks;
    a.window = p->window;
    a.sink = p->sink;
    a.scale_log2 = (float)((double)p->scale * 1.4426950408889634);
    return launched(kv4_attn(a, f16, plan, p->work, st), who);
}

}  // extern "C"
