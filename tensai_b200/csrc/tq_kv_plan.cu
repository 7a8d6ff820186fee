// tq_kv_plan.cu — the bookkeeping of a paged cache on the GPU: block tables,
// slots and the free list from the lengths of the requests (tq_kv_plan_dev,
// tq_kv_release_dev).
//
// With have_i = ceil(cached_i / P) and want_i = ceil((cached_i + added_i) / P)
// the new pages of request i are numbers F_i .. F_i + want_i - have_i - 1 of the
// call, F the exclusive sums of want - have, and its new tokens are numbers
// S_i .. S_i + added_i - 1, S the exclusive sums of added. Both sums are made
// by every block in its own shared memory (8 bytes read per request), after
// which each new table entry and each slot is found on its own by a binary
// search in them: no block waits for another's results.
//
// One launch of one cluster of 1 to 8 blocks: the blocks share the entries and
// slots evenly, and the cluster's barrier separates all reads of the lengths
// (into every block's shared memory) and the free count from their updates in
// place, so a graph that holds the step can be replayed without a copy of either.
//
// The ids that a call would take are looked at before it writes anything (0.3 us
// for 8 requests, 0.9 for 1,024: it changes nothing if one is outside the cache).
//
// Bound by latency: the launch, three dependent loads, two scans, the searches.
// In a graph 8 requests take 3.7 us; 1,024 requests with 54,290 new tokens 10.7
// us (0.48 MB), with a cluster of four blocks 16.0, with one block 43.0.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <climits>

#include "tq_common.cuh"
#include "tq_kv.h"

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 1024;
constexpr int kMaxCluster = 8;
constexpr int kSide = 4; // slots that a thread finds side by side

// For each of B values x: the largest i < n with sums[i] <= x, for ascending
// sums[0] = 0 .. sums[n] > x; the B searches run side by side.
template <int B> __device__ __forceinline__ void find_rows(const int *sums, int n, const int (&x)[B], int (&row)[B]) {
#pragma unroll
    for (int u = 0; u < B; u++) row[u] = 0;
    for (int step = 1 << (31 - __clz(n)); step; step >>= 1)
#pragma unroll
        for (int u = 0; u < B; u++) {
            const int at = row[u] + step;
            if (at < n && sums[at] <= x[u]) row[u] = at;
        }
}

// The or of every thread's bits, to all of them. *sh: zero before a barrier that precedes the call.
__device__ __forceinline__ unsigned block_or(unsigned bits, unsigned *sh) {
    if (bits) atomicOr(sh, bits);
    __syncthreads();
    return *sh;
}

// Exclusive sums over the block of a (64 bits) and b per thread; the totals in *ta, *tb.
__device__ __forceinline__ void block_scan(long long &a, long long &b, long long *ta, long long *tb) {
    __shared__ long long wa[32], wb[32];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    long long ia = a, ib = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long ua = __shfl_up_sync(0xffffffffu, ia, o), ub = __shfl_up_sync(0xffffffffu, ib, o);
        if (lane >= o) ia += ua, ib += ub;
    }
    if (lane == 31) wa[w] = ia, wb[w] = ib;
    __syncthreads();
    if (w == 0) {
        long long va = wa[lane], vb = wb[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long ua = __shfl_up_sync(0xffffffffu, va, o), ub = __shfl_up_sync(0xffffffffu, vb, o);
            if (lane >= o) va += ua, vb += ub;
        }
        wa[lane] = va, wb[lane] = vb;
    }
    __syncthreads();
    a = ia - a + (w ? wa[w - 1] : 0);
    b = ib - b + (w ? wb[w - 1] : 0);
    *ta = wa[31], *tb = wb[31];
}

__global__ void __launch_bounds__(kThreads) kv_plan_kernel(tq_kv_plan_args a, int shift, int n_pages, unsigned *status) {
    extern __shared__ int sums[]; // [n + 1] token starts, [n + 1] new-page starts, [n] cached
    int *tok = sums, *pag = sums + a.n + 1, *held = pag + a.n + 1;
    __shared__ unsigned s_bad;
    const int n = a.n, tid = threadIdx.x, P = 1 << shift;
    cg::cluster_group cl = cg::this_cluster();
    const int rank = (int)cl.block_rank(), blocks = (int)cl.num_blocks();
    const int per = (n + kThreads - 1) / kThreads, i0 = min(n, tid * per), i1 = min(n, i0 + per);
    const int count = *a.free_count;
    if (tid == 0) s_bad = 0;
    long long st = 0, sp = 0;
    unsigned bad = 0;
    for (int i = i0; i < i1; i++) {
        const int ci = a.cached[i], di = a.added[i];
        held[i] = ci;
        tok[i] = di; // until the sums are known
        const long long c = ci, d = di, have = (c + P - 1) >> shift, want = (c + d + P - 1) >> shift;
        if (c < 0 || d < 0 || c + d > INT_MAX) bad |= TQ_KV_STATUS_LENGTH;
        if (want > a.table_cols) bad |= TQ_KV_STATUS_TABLE;
        st += d;
        sp += want - have;
    }
    long long tokens, pages;
    block_scan(st, sp, &tokens, &pages);
    if (tokens > a.slots_cap) bad |= TQ_KV_STATUS_SLOTS;
    if (count < 0 || count > a.free_cap) bad |= TQ_KV_STATUS_LENGTH;
    if (pages > count) bad |= TQ_KV_STATUS_POOL;
    if (count <= a.free_cap && pages <= count) // the ids that the call would take; read again below, near by then
        for (int j = tid; j < (int)pages; j += kThreads) {
            const int id = a.free_pages[count - 1 - j];
            if (id < 0 || id >= n_pages) bad |= TQ_KV_STATUS_PAGE;
        }
    bad = block_or(bad, &s_bad); // one verdict for the block; every block of the cluster reaches the same one
    if (blocks > 1) cl.barrier_arrive(); // this block has read what may be written in place
    const int g = rank * kThreads + tid, stride = blocks * kThreads;
    if (bad) {
        if (g == 0) atomicOr(status, bad);
        for (int i = g; i <= n; i += stride) a.starts[i] = 0;
        for (int t = g; t < a.slots_cap; t += stride) a.slots[t] = -1;
        if (blocks > 1) cl.barrier_wait();
        for (int i = g; i < n; i += stride) a.lens[i] = held[i];
        if (g == 0) *a.free_left = count;
        return;
    }
    for (int i = i0; i < i1; i++) {
        const int c = held[i], d = tok[i];
        tok[i] = (int)st;
        pag[i] = (int)sp;
        st += d;
        sp += ((c + d + P - 1) >> shift) - ((c + P - 1) >> shift);
    }
    if (tid == 0) tok[n] = (int)tokens, pag[n] = (int)pages;
    __syncthreads();
    for (int i = g; i <= n; i += stride) a.starts[i] = tok[i];
    for (int j0 = g; j0 < (int)pages; j0 += stride) { // new table entries
        const int j[1] = {j0}, id = a.free_pages[count - 1 - j0];
        int i[1];
        find_rows(pag, n, j, i);
        a.table[(size_t)i[0] * a.table_stride + ((held[i[0]] + P - 1) >> shift) + (j0 - pag[i[0]])] = id;
    }
    for (int t0 = g; t0 < (int)tokens; t0 += kSide * stride) { // slots
        int t[kSide], i[kSide], pos[kSide], id[kSide];
#pragma unroll
        for (int u = 0; u < kSide; u++) t[u] = min(t0 + u * stride, (int)tokens - 1);
        find_rows(tok, n, t, i);
#pragma unroll
        for (int u = 0; u < kSide; u++) {
            const int c = held[i[u]], have = (c + P - 1) >> shift;
            pos[u] = c + (t[u] - tok[i[u]]);
            const int b = pos[u] >> shift;
            id[u] = b >= have ? a.free_pages[count - 1 - pag[i[u]] - (b - have)] : a.table[(size_t)i[u] * a.table_stride + b];
        }
#pragma unroll
        for (int u = 0; u < kSide; u++) {
            const bool ok = id[u] >= 0 && id[u] < n_pages;
            if (!ok) atomicOr(status, TQ_KV_STATUS_PAGE);
            if (t0 + u * stride < (int)tokens) a.slots[t[u]] = ok ? ((long long)id[u] << shift) + (pos[u] & (P - 1)) : -1;
        }
    }
    if (blocks > 1) cl.barrier_wait();
    for (int i = g; i < n; i += stride) a.lens[i] = held[i] + (tok[i + 1] - tok[i]);
    if (g == 0) *a.free_left = count - (int)pages;
}

__global__ void __launch_bounds__(kThreads) kv_release_kernel(tq_kv_release_args a, int shift, int n_pages,
                                                              unsigned *status) {
    extern __shared__ int sums[]; // [n + 1] page starts of the released requests
    __shared__ unsigned s_bad_id;
    const int n = a.n, tid = threadIdx.x, P = 1 << shift;
    const int per = (n + kThreads - 1) / kThreads, i0 = min(n, tid * per), i1 = min(n, i0 + per);
    const int count = *a.free_count;
    long long sp = 0, none = 0, pages, unused;
    __shared__ unsigned s_bad;
    if (tid == 0) s_bad = s_bad_id = 0;
    unsigned bad = 0;
    for (int i = i0; i < i1; i++) {
        if (!a.done[i]) continue;
        const long long have = ((long long)a.lens[i] + P - 1) >> shift;
        if (a.lens[i] < 0) bad |= TQ_KV_STATUS_LENGTH;
        if (have > a.table_cols) bad |= TQ_KV_STATUS_TABLE;
        sp += have;
    }
    block_scan(sp, none, &pages, &unused);
    if (count < 0 || count > a.free_cap) bad |= TQ_KV_STATUS_LENGTH;
    if (count + pages > a.free_cap) bad |= TQ_KV_STATUS_POOL;
    bad = block_or(bad, &s_bad);
    auto refuse = [&]() {
        if (tid == 0) {
            atomicOr(status, bad);
            *a.free_left = count;
        }
    };
    if (bad) return refuse();
    for (int i = i0; i < i1; i++) {
        sums[i] = (int)sp;
        if (a.done[i]) sp += (a.lens[i] + P - 1) >> shift;
    }
    if (tid == 0) sums[n] = (int)pages;
    __syncthreads();
    auto page = [&](int j) { // the j-th released page
        const int x[1] = {j};
        int i[1];
        find_rows(sums, n, x, i);
        return a.table[(size_t)i[0] * a.table_stride + (j - sums[i[0]])];
    };
    for (int j = tid; j < (int)pages; j += kThreads) {
        const int id = page(j);
        if (id < 0 || id >= n_pages) bad |= TQ_KV_STATUS_PAGE;
    }
    bad = block_or(bad, &s_bad_id);
    if (bad) return refuse();
    for (int j = tid; j < (int)pages; j += kThreads) a.free_pages[count + j] = page(j);
    for (int i = tid; i < n; i += kThreads)
        if (a.done[i]) a.lens[i] = 0;
    if (tid == 0) *a.free_left = count + (int)pages;
}

__global__ void kv_take_kernel(unsigned *status, unsigned *bits) { *bits = atomicExch(status, 0u); }

TqDeviceOnce g_once;

cudaError_t set_up() {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    return tq_device_once(g_once, dev, [] {
        const int most = 3 * (TQ_KV_MAX_REQUESTS + 1) * (int)sizeof(int);
        cudaError_t r = cudaFuncSetAttribute(kv_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        if (r == cudaSuccess)
            r = cudaFuncSetAttribute(kv_release_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most / 3);
        return r;
    });
}

} // namespace

cudaError_t tq_kv_launch_plan(int page_shift, int n_pages, unsigned *status, const tq_kv_plan_args &a, cudaStream_t st) {
    cudaError_t e = set_up();
    if (e != cudaSuccess) return e;
    // As many blocks as have 2048 requests and slots each (256 each measured the same).
    const long long work = (long long)a.n + a.slots_cap;
    int blocks = 1;
    while (blocks < kMaxCluster && work > (long long)blocks * 2 * kThreads) blocks *= 2;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = blocks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = 3 * (size_t)(a.n + 1) * sizeof(int);
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kv_plan_kernel, a, page_shift, n_pages, status);
}

cudaError_t tq_kv_launch_take(unsigned *status, unsigned *bits, cudaStream_t st) {
    kv_take_kernel<<<1, 1, 0, st>>>(status, bits);
    return cudaGetLastError();
}

cudaError_t tq_kv_launch_release(int page_shift, int n_pages, unsigned *status, const tq_kv_release_args &a,
                                 cudaStream_t st) {
    cudaError_t e = set_up();
    if (e != cudaSuccess) return e;
    kv_release_kernel<<<1, kThreads, (size_t)(a.n + 1) * sizeof(int), st>>>(a, page_shift, n_pages, status);
    return cudaGetLastError();
}
