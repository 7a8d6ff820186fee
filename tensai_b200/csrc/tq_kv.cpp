// tq_kv.cpp — the tq_kv_* entry points: cache handles, argument checks and
// dispatch to the kernels (tq_kv_plan.cu, tq_kv_store.cu, tq_kv_attn.cu). Every
// call runs on the cache's device and leaves the thread's current device as it
// was.
#include <cuda_runtime.h>

#include <climits>
#include <cmath>
#include <cstring>
#include <initializer_list>
#include <memory>
#include <mutex>
#include <new>
#include <shared_mutex>
#include <unordered_map>
#include <vector>

#include "../../include/tensai_cuda.h"
#include "tq_internal.h"
#include "tq_kv.h"

namespace {

struct KvCache {
    int device = 0, hdp = 0, shift = 0, sms = 0;
    tq_kv_config c{};
    std::vector<TqKvLayer> layers;
    unsigned *status = nullptr; // TQ_KV_STATUS_* bits, then those last looked at
    std::mutex look;            // one look at a time
    std::shared_mutex use;      // held by every call up to its last launch; by tq_kv_free alone
    bool freed = false;
    std::mutex launch; // an attention's launches follow one another: threads may share a stream and a workspace
};

std::mutex g_kv_mu;
std::unordered_map<uint64_t, std::shared_ptr<KvCache>> g_caches;
uint64_t g_next_cache = 1;

// The cache's device for the length of a call.
struct OnDevice {
    int prev = -1;
    cudaError_t err;
    explicit OnDevice(int device) {
        err = cudaGetDevice(&prev);
        if (err == cudaSuccess && prev != device)
            err = cudaSetDevice(device);
        else
            prev = -1;
    }
    ~OnDevice() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};

void release(KvCache &k) {
    for (TqKvLayer &l : k.layers)
        for (void *p : {(void *)l.k, (void *)l.v, (void *)l.scale})
            if (p) cudaFree(p);
    k.layers.clear();
    if (k.status) cudaFree(k.status);
    k.status = nullptr;
}

// A cache in use by a call: its memory stays until the call has made its launches.
struct InUse {
    std::shared_ptr<KvCache> k; // destroyed after the lock
    std::shared_lock<std::shared_mutex> lk;
    explicit operator bool() const { return k != nullptr; }
    KvCache *operator->() const { return k.get(); }
    KvCache &operator*() const { return *k; }
};
InUse find(uint64_t h, int *rc) {
    InUse u;
    *rc = TQ_OK;
    {
        std::lock_guard<std::mutex> lk(g_kv_mu);
        auto it = g_caches.find(h);
        if (it != g_caches.end()) u.k = it->second;
    }
    if (u) {
        u.lk = std::shared_lock<std::shared_mutex>(u->use);
        if (!u->freed) return u;
        u.lk.unlock();
        u.k.reset();
    }
    *rc = tq_fail(TQ_ERR_HANDLE, "tensai: invalid or freed cache handle %llu", (unsigned long long)h);
    return u;
}

TqKvView view(const KvCache &k, int layer) {
    const TqKvLayer &l = k.layers[layer];
    return {l.k, l.v, l.scale, k.status, k.c.n_kv, k.c.hd, k.hdp, k.c.page, k.shift, k.c.n_pages};
}

int check_layer(const KvCache &k, int layer) {
    if (layer >= 0 && layer < k.c.n_layer) return TQ_OK;
    return tq_fail(TQ_ERR_ARG, "tensai: cache layer %d out of range [0, %d)", layer, k.c.n_layer);
}

int check_dtype(int dtype) {
    if (dtype == TQ_LINEAR_F32 || dtype == TQ_LINEAR_F16 || dtype == TQ_LINEAR_BF16) return TQ_OK;
    return tq_fail(TQ_ERR_ARG, "tensai: unknown cache element type %d", dtype);
}

size_t size_of(int dtype) { return dtype == TQ_LINEAR_F32 ? 4 : 2; }

bool overlap(const void *a, size_t na, const void *b, size_t nb) {
    const char *x = static_cast<const char *>(a), *y = static_cast<const char *>(b);
    return na && nb && x < y + nb && y < x + na;
}

// Whether every pointer is a multiple of `to`, which the kernels' accesses rely on.
bool aligned(std::initializer_list<const void *> ps, size_t to) {
    for (const void *p : ps)
        if ((uintptr_t)p % to) return false;
    return true;
}
int unaligned(const char *what) {
    return tq_fail(TQ_ERR_ARG, "tensai: %s not aligned to their type", what);
}

// Indexes in the kernels are int: a position, token or row may be stepped past by a
// tile, a window or the threads of a cluster, and stays one.
constexpr int kMostIndex = INT_MAX - 65536;

int check_table(const KvCache &k, const char *what, int cols, int stride) {
    if (cols < 0 || stride < cols)
        return tq_fail(TQ_ERR_ARG, "tensai: bad %s table: rows of %d in %d", what, cols, stride);
    if (cols > kMostIndex / k.c.page)
        return tq_fail(TQ_ERR_UNSUPPORTED, "tensai: %s table rows of %d pages of %d tokens are too long", what, cols,
                       k.c.page);
    return TQ_OK;
}
int check_most(const char *what, long long n) {
    if (n <= kMostIndex) return TQ_OK;
    return tq_fail(TQ_ERR_UNSUPPORTED, "tensai: %lld %s in one call, at most %d", n, what, kMostIndex);
}

int bad_pages(const char *what, int n) {
    return tq_fail(TQ_ERR_ARG, "tensai: %s of %d pages: null pointer or negative count", what, n);
}

int done(cudaError_t e, const char *what) { return e == cudaSuccess ? TQ_OK : tq_cuda_fail(e, what); }

} // namespace

extern "C" {

int tq_kv_create(const tq_kv_config *cfg, uint64_t *cache) {
    if (!cfg || !cache) return tq_fail(TQ_ERR_ARG, "tensai: null pointer argument");
    const tq_kv_config &c = *cfg;
    if (c.n_layer < 1 || c.n_kv < 1 || c.n_pages < 1 || c.n_kv > 65535 || c.n_layer > 65535)
        return tq_fail(TQ_ERR_ARG, "tensai: a cache needs layers, KV heads (at most 65535 each) and pages, got %d, %d, %d",
                       c.n_layer, c.n_kv, c.n_pages);
    if (c.hd < 8 || c.hd > 256 || c.hd % 8)
        return tq_fail(TQ_ERR_ARG, "tensai: cache head size must be a multiple of 8 up to 256, got %d", c.hd);
    if (c.page != 16 && c.page != 32 && c.page != 64 && c.page != 128)
        return tq_fail(TQ_ERR_ARG, "tensai: cache pages hold 16, 32, 64 or 128 tokens, got %d", c.page);
    std::shared_ptr<KvCache> k;
    try {
        k = std::make_shared<KvCache>();
        k->layers.resize(c.n_layer);
    } catch (const std::bad_alloc &) {
        return tq_fail(TQ_ERR_NOMEM, "tensai: out of host memory for a cache of %d layers", c.n_layer);
    }
    k->c = c;
    k->hdp = c.hd <= 64 ? 64 : c.hd <= 128 ? 128 : 256;
    for (k->shift = 4; (1 << k->shift) < c.page;) k->shift++;
    const unsigned __int128 bytes = (unsigned __int128)c.n_pages * c.n_kv * c.page * k->hdp;
    if (bytes > ((unsigned __int128)1 << 46))
        return tq_fail(TQ_ERR_UNSUPPORTED, "tensai: a cache of %d pages is too large", c.n_pages);
    const size_t codes = (size_t)bytes, scales = (size_t)c.n_pages * c.n_kv * sizeof(float2);
    cudaError_t e = cudaGetDevice(&k->device);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&k->sms, cudaDevAttrMultiProcessorCount, k->device);
    if (e == cudaSuccess) e = tq_dev_malloc((void **)&k->status, 2 * sizeof(unsigned));
    if (e == cudaSuccess) e = cudaMemset(k->status, 0, 2 * sizeof(unsigned));
    for (TqKvLayer &l : k->layers) {
        if (e == cudaSuccess) e = tq_dev_malloc((void **)&l.k, codes);
        if (e == cudaSuccess) e = tq_dev_malloc((void **)&l.v, codes);
        if (e == cudaSuccess) e = tq_dev_malloc((void **)&l.scale, scales);
        if (e == cudaSuccess) e = cudaMemset(l.k, TQ_KV_ZERO, codes);
        if (e == cudaSuccess) e = cudaMemset(l.v, TQ_KV_ZERO, codes);
        if (e == cudaSuccess) e = cudaMemset(l.scale, 0, scales);
    }
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    if (e != cudaSuccess) {
        release(*k);
        return tq_cuda_fail(e, "cache allocation");
    }
    try {
        std::lock_guard<std::mutex> lk(g_kv_mu);
        g_caches.emplace(g_next_cache, k);
        *cache = g_next_cache++;
    } catch (const std::bad_alloc &) {
        release(*k);
        return tq_fail(TQ_ERR_NOMEM, "tensai: out of host memory for a cache handle");
    }
    return TQ_OK;
}

int tq_kv_free(uint64_t cache) {
    std::shared_ptr<KvCache> k;
    {
        std::lock_guard<std::mutex> lk(g_kv_mu);
        auto it = g_caches.find(cache);
        if (it == g_caches.end()) return TQ_OK;
        k = it->second;
        g_caches.erase(it);
    }
    std::lock_guard<std::shared_mutex> lk(k->use); // calls of other threads have made their launches
    k->freed = true;
    OnDevice on(k->device);
    cudaDeviceSynchronize(); // no kernel of any stream may still read the pages
    release(*k);
    return TQ_OK;
}

int tq_kv_info(uint64_t cache, tq_kv_config *cfg, int *device) {
    int rc;
    auto k = find(cache, &rc);
    if (!k) return rc;
    if (cfg) *cfg = k->c;
    if (device) *device = k->device;
    return TQ_OK;
}

int tq_kv_status(uint64_t cache, unsigned *bits) {
    if (!bits) return tq_fail(TQ_ERR_ARG, "tensai: null output pointer");
    *bits = 0;
    int rc;
    auto k = find(cache, &rc);
    if (!k) return rc;
    OnDevice on(k->device);
    cudaError_t e = on.err;
    std::lock_guard<std::mutex> lk(k->look);
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    if (e == cudaSuccess) e = tq_kv_launch_take(k->status, k->status + 1, nullptr);
    if (e == cudaSuccess) e = cudaMemcpy(bits, k->status + 1, sizeof *bits, cudaMemcpyDeviceToHost);
    return done(e, "cache status");
}

int tq_kv_plan_dev(uint64_t cache, const tq_kv_plan_args *args, void *stream) {
    int rc;
    auto k = find(cache, &rc);
    if (!k) return rc;
    if (!args) return tq_fail(TQ_ERR_ARG, "tensai: null pointer argument");
    const tq_kv_plan_args &a = *args;
    if (a.n < 0 || a.n > TQ_KV_MAX_REQUESTS)
        return tq_fail(a.n < 0 ? TQ_ERR_ARG : TQ_ERR_UNSUPPORTED, "tensai: a plan takes 0 to %d requests, got %d",
                       TQ_KV_MAX_REQUESTS, a.n);
    if (a.slots_cap < 0 || a.free_cap < 0)
        return tq_fail(TQ_ERR_ARG, "tensai: bad plan sizes: %d slots, %d free pages", a.slots_cap, a.free_cap);
    if ((rc = check_table(*k, "plan", a.table_cols, a.table_stride)) || (rc = check_most("slots", a.slots_cap)) ||
        (rc = check_most("free pages", a.free_cap)))
        return rc;
    if ((a.n && (!a.cached || !a.added || !a.lens || (!a.table && a.table_cols))) || !a.starts || !a.free_count ||
        !a.free_left || (a.free_cap && !a.free_pages) || (a.slots_cap && !a.slots))
        return tq_fail(TQ_ERR_ARG, "tensai: null pointer argument");
    if (!aligned({a.cached, a.added, a.table, a.free_pages, a.free_count, a.starts, a.lens, a.free_left}, sizeof(int)) ||
        !aligned({a.slots}, sizeof(long long)))
        return unaligned("plan arrays");
    const size_t n4 = sizeof(int) * (size_t)a.n;
    const struct {
        const void *p;
        size_t bytes;
    } in[] = {{a.cached, n4}, {a.added, n4}, {a.free_pages, sizeof(int) * (size_t)a.free_cap}, {a.free_count, sizeof(int)}},
      out[] = {{a.starts, n4 + sizeof(int)},
               {a.lens, n4},
               {a.slots, sizeof(long long) * (size_t)a.slots_cap},
               {a.table, a.n ? sizeof(int) * ((size_t)a.table_stride * (a.n - 1) + a.table_cols) : 0},
               {a.free_left, sizeof(int)}};
    for (size_t i = 0; i < sizeof out / sizeof *out; i++) {
        for (const auto &x : in) {
            const bool in_place = (out[i].p == a.lens && x.p == a.cached && a.lens == a.cached) ||
                                  (out[i].p == a.free_left && x.p == a.free_count && a.free_left == a.free_count);
            if (!in_place && overlap(out[i].p, out[i].bytes, x.p, x.bytes))
                return tq_fail(TQ_ERR_ARG, "tensai: plan arrays overlap");
        }
        for (size_t j = 0; j < i; j++)
            if (overlap(out[i].p, out[i].bytes, out[j].p, out[j].bytes))
                return tq_fail(TQ_ERR_ARG, "tensai: plan arrays overlap");
    }
    OnDevice on(k->device);
    if (on.err != cudaSuccess) return tq_cuda_fail(on.err, "set device");
    return done(tq_kv_launch_plan(k->shift, k->c.n_pages, k->status, a, (cudaStream_t)stream), "plan launch");
}

int tq_kv_release_dev(uint64_t cache, const tq_kv_release_args *args, void *stream) {
    int rc;
    auto k = find(cache, &rc);
    if (!k) return rc;
    if (!args) return tq_fail(TQ_ERR_ARG, "tensai: null pointer argument");
    const tq_kv_release_args &a = *args;
    if (a.n < 0 || a.n > TQ_KV_MAX_REQUESTS)
        return tq_fail(a.n < 0 ? TQ_ERR_ARG : TQ_ERR_UNSUPPORTED, "tensai: a release takes 0 to %d requests, got %d",
                       TQ_KV_MAX_REQUESTS, a.n);
    if (a.free_cap < 0) return tq_fail(TQ_ERR_ARG, "tensai: bad release sizes: %d free pages", a.free_cap);
    if ((rc = check_table(*k, "release", a.table_cols, a.table_stride)) || (rc = check_most("free pages", a.free_cap)))
        return rc;
    if ((a.n && (!a.done || !a.lens || (!a.table && a.table_cols))) || !a.free_count || !a.free_left ||
        (a.free_cap && !a.free_pages))
        return tq_fail(TQ_ERR_ARG, "tensai: null pointer argument");
    if (!aligned({a.done, a.lens, a.table, a.free_pages, a.free_count, a.free_left}, sizeof(int)))
        return unaligned("release arrays");
    const size_t n4 = sizeof(int) * (size_t)a.n, fb = sizeof(int) * (size_t)a.free_cap,
                 tb = a.n ? sizeof(int) * ((size_t)a.table_stride * (a.n - 1) + a.table_cols) : 0;
    if (overlap(a.lens, n4, a.done, n4) || overlap(a.lens, n4, a.table, tb) || overlap(a.lens, n4, a.free_pages, fb) ||
        overlap(a.lens, n4, a.free_left, 4) || overlap(a.lens, n4, a.free_count, 4) ||
        overlap(a.free_pages, fb, a.done, n4) || overlap(a.free_pages, fb, a.table, tb) ||
        overlap(a.free_pages, fb, a.free_left, 4) || overlap(a.free_pages, fb, a.free_count, 4) ||
        overlap(a.free_left, 4, a.done, n4) || overlap(a.free_left, 4, a.table, tb) ||
        (a.free_left != a.free_count && overlap(a.free_left, 4, a.free_count, 4)))
        return tq_fail(TQ_ERR_ARG, "tensai: release arrays overlap");
    OnDevice on(k->device);
    if (on.err != cudaSuccess) return tq_cuda_fail(on.err, "set device");
    return done(tq_kv_launch_release(k->shift, k->c.n_pages, k->status, a, (cudaStream_t)stream), "release launch");
}

int tq_kv_store_dev(uint64_t cache, int layer, const void *k, const void *v, int dtype, long long k_stride,
                    long long v_stride, const long long *slots, int n, void *stream) {
    int rc;
    auto c = find(cache, &rc);
    if (!c || (rc = check_layer(*c, layer)) || (rc = check_dtype(dtype))) return rc;
    const long long row = (long long)c->c.n_kv * c->c.hd;
    if (n < 0) return tq_fail(TQ_ERR_ARG, "tensai: negative token count %d", n);
    if ((rc = check_most("tokens", n))) return rc;
    if (n && (!k || !v || !slots)) return tq_fail(TQ_ERR_ARG, "tensai: null pointer argument");
    if (n > 1 && (k_stride < row || v_stride < row))
        return tq_fail(TQ_ERR_ARG, "tensai: key and value rows of %lld elements do not fit strides of %lld and %lld",
                       row, k_stride, v_stride);
    if (!aligned({k, v}, size_of(dtype)) || !aligned({slots}, sizeof(long long)))
        return unaligned("keys, values or slots");
    OnDevice on(c->device);
    if (on.err != cudaSuccess) return tq_cuda_fail(on.err, "set device");
    return done(tq_kv_launch_store(view(*c, layer), k, v, dtype, k_stride, v_stride, slots, n, c->sms, (cudaStream_t)stream),
                "cache store launch");
}

int tq_kv_attention_workspace(uint64_t cache, size_t *bytes) {
    if (!bytes) return tq_fail(TQ_ERR_ARG, "tensai: null output pointer");
    *bytes = 0;
    int rc;
    auto k = find(cache, &rc);
    if (!k) return rc;
    *bytes = tq_kv_attn_workspace(k->hdp, k->sms);
    return TQ_OK;
}

int tq_kv_attention_dev(uint64_t cache, int layer, const tq_kv_attention_args *args, void *stream) {
    int rc;
    auto k = find(cache, &rc);
    if (!k || (rc = check_layer(*k, layer))) return rc;
    if (!args) return tq_fail(TQ_ERR_ARG, "tensai: null pointer argument");
    const tq_kv_attention_args &a = *args;
    if ((rc = check_dtype(a.dtype))) return rc;
    if (a.n_q < 1 || a.n_q % k->c.n_kv)
        return tq_fail(TQ_ERR_ARG, "tensai: %d query heads do not share %d KV heads evenly", a.n_q, k->c.n_kv);
    if (a.n < 0 || a.n > TQ_KV_MAX_REQUESTS || a.n_tokens < 0)
        return tq_fail(a.n > TQ_KV_MAX_REQUESTS ? TQ_ERR_UNSUPPORTED : TQ_ERR_ARG,
                       "tensai: attention takes 0 to %d sequences, got %d (of %d tokens)", TQ_KV_MAX_REQUESTS, a.n,
                       a.n_tokens);
    const long long row = (long long)a.n_q * k->c.hd;
    if ((rc = check_most("rows (tokens x query heads)", (long long)a.n_tokens * a.n_q))) return rc;
    if (a.n_tokens > 1 && (a.q_stride < row || a.out_stride < row))
        return tq_fail(TQ_ERR_ARG, "tensai: query rows of %lld elements do not fit strides of %lld and %lld", row,
                       a.q_stride, a.out_stride);
    if ((rc = check_table(*k, "attention", a.table_cols, a.table_stride))) return rc;
    if (!std::isfinite(a.scale)) return tq_fail(TQ_ERR_ARG, "tensai: attention scale is not finite");
    if (a.n == 0 || a.n_tokens == 0) return TQ_OK;
    if (!a.q || !a.out || !a.starts || !a.lens || (!a.table && a.table_cols) || !a.workspace)
        return tq_fail(TQ_ERR_ARG, "tensai: null pointer argument");
    if (!aligned({a.q, a.out}, size_of(a.dtype)) || !aligned({a.starts, a.lens, a.table}, sizeof(int)))
        return unaligned("queries, outputs, lengths or tables");
    const size_t span_q = size_of(a.dtype) * ((size_t)a.q_stride * (a.n_tokens - 1) + row),
                 span_o = size_of(a.dtype) * ((size_t)a.out_stride * (a.n_tokens - 1) + row);
    if (overlap(a.q, span_q, a.out, span_o)) return tq_fail(TQ_ERR_ARG, "tensai: attention output overlaps its queries");
    const size_t need = tq_kv_attn_workspace(k->hdp, k->sms);
    if (a.workspace_bytes < need || (uintptr_t)a.workspace % 16)
        return tq_fail(TQ_ERR_ARG, "tensai: attention needs a 16-byte aligned workspace of %zu bytes, got %zu", need,
                       a.workspace_bytes);
    if (overlap(a.workspace, need, a.out, span_o) || overlap(a.workspace, need, a.q, span_q))
        return tq_fail(TQ_ERR_ARG, "tensai: attention workspace overlaps its queries or output");
    OnDevice on(k->device);
    if (on.err != cudaSuccess) return tq_cuda_fail(on.err, "set device");
    const TqKvAttn t = {a.q,      a.out,  a.dtype, a.q_stride,     a.out_stride, a.n_q,   a.n_tokens,
                        a.n,      a.starts, a.lens, a.table,       a.table_stride, a.table_cols, a.scale, a.workspace};
    std::lock_guard<std::mutex> lk(k->launch);
    return done(tq_kv_launch_attn(view(*k, layer), t, k->sms, (cudaStream_t)stream), "attention launch");
}

int tq_kv_load_dev(uint64_t cache, int layer, const int *pages, int n, const int8_t *k, const int8_t *v,
                   const float *kscale, const float *vscale, void *stream) {
    int rc;
    auto c = find(cache, &rc);
    if (!c || (rc = check_layer(*c, layer))) return rc;
    if (n < 0 || (n && (!pages || !k || !v || !kscale || !vscale))) return bad_pages("load", n);
    if (!aligned({k, v}, 4)) return tq_fail(TQ_ERR_ARG, "tensai: codes must be 4-byte aligned");
    if (!aligned({pages, kscale, vscale}, sizeof(int))) return unaligned("pages or scales");
    OnDevice on(c->device);
    if (on.err != cudaSuccess) return tq_cuda_fail(on.err, "set device");
    return done(tq_kv_launch_load(view(*c, layer), pages, n, k, v, kscale, vscale, (cudaStream_t)stream),
                "cache load launch");
}

int tq_kv_save_dev(uint64_t cache, int layer, const int *pages, int n, int8_t *k, int8_t *v, float *kscale,
                   float *vscale, void *stream) {
    int rc;
    auto c = find(cache, &rc);
    if (!c || (rc = check_layer(*c, layer))) return rc;
    if (n < 0 || (n && (!pages || !k || !v || !kscale || !vscale))) return bad_pages("save", n);
    if (!aligned({k, v}, 4)) return tq_fail(TQ_ERR_ARG, "tensai: codes must be 4-byte aligned");
    if (!aligned({pages, kscale, vscale}, sizeof(int))) return unaligned("pages or scales");
    OnDevice on(c->device);
    if (on.err != cudaSuccess) return tq_cuda_fail(on.err, "set device");
    return done(tq_kv_launch_save(view(*c, layer), pages, n, k, v, kscale, vscale, (cudaStream_t)stream),
                "cache save launch");
}

int tq_kv_read_dev(uint64_t cache, int layer, const int *pages, int n, float *k, float *v, void *stream) {
    int rc;
    auto c = find(cache, &rc);
    if (!c || (rc = check_layer(*c, layer))) return rc;
    if (n < 0 || (n && (!pages || !k || !v))) return bad_pages("read", n);
    if (!aligned({k, v}, 16)) return tq_fail(TQ_ERR_ARG, "tensai: values must be 16-byte aligned");
    if (!aligned({pages}, sizeof(int))) return unaligned("pages");
    OnDevice on(c->device);
    if (on.err != cudaSuccess) return tq_cuda_fail(on.err, "set device");
    return done(tq_kv_launch_read(view(*c, layer), pages, n, k, v, (cudaStream_t)stream), "cache read launch");
}

} // extern "C"
