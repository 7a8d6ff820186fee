// tq_kv_store.cu — new keys and values into the paged 8-bit cache, and pages
// of it in and out (tq_kv_store_dev, tq_kv_load_dev, tq_kv_save_dev,
// tq_kv_read_dev; layout in tq_kv.h).
//
// One block per run of tokens that share a page, KV head and side (keys or
// values): it alone reads and writes that page's codes and scale, so there are
// no atomics and the result does not depend on timing. It
//   reads the run into shared memory once and takes max|x| (as an integer
//   maximum of the encodings, which keeps a NaN);
//   scale = float32(max / 127), at least the present scale when the page holds
//   earlier positions, whose codes are rounded again if the scale grew;
//   rounds x / scale to the nearest integer, ties to even, of the exact
//   quotient: the product with 1 / scale decides it except within 1e-4 of a
//   half, where the sign of x - (t + 1/2) scale, exact in one FMA, does. (A
//   plain float division puts about one value in 10^5 on the wrong side.)
// Bound by HBM at prompt sizes (element in, byte out), by latency in a decode
// step.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "tq_common.cuh"
#include "tq_kv.h"

namespace {

constexpr int kStoreThreads = 128;
constexpr int kMaxPage = 128;
static_assert(kStoreThreads >= kMaxPage, "one thread per token of a run");

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }

// The integer nearest to x / s (ties to even), |x| <= 127 s up to rounding.
__device__ __forceinline__ int code_of(float x, float s, float inv) {
    if (!(s > 0.f)) return 0; // zero or NaN
    if (s < 0x1p-100f)        // the products below could underflow
        return (int)fmin(fmax(rint(__ddiv_rn((double)x, (double)s)), -127.0), 127.0);
    const float y = __fmul_rn(x, inv);
    float t = rintf(y);
    if (fabsf(y - t) > 0.4999f) {
        const float lo = floorf(y); // the half between lo and lo + 1 decides
        const float r = __fmaf_rn(-(lo + 0.5f), s, x);
        t = r > 0.f ? lo + 1.f : r < 0.f ? lo : 2.f * rintf(0.5f * (lo + 0.5f));
    }
    return (int)fminf(fmaxf(t, -127.f), 127.f);
}

// The integer nearest to c * was / now (ties to even).
__device__ __forceinline__ int recode(int c, float was, float now, float ratio) {
    const float y = __fmul_rn((float)c, ratio), t = rintf(y);
    if (fabsf(y - t) > 0.4999f) return (int)rint(__ddiv_rn((double)c * (double)was, (double)now));
    return (int)t;
}

__device__ __forceinline__ unsigned byte_of(unsigned w, int i) { return (w >> (8 * i)) & 0xffu; }

template <typename T, bool VEC>
__global__ void __launch_bounds__(kStoreThreads) kv_store_kernel(TqKvView c, const T *k, const T *v, long long k_stride,
                                                                 long long v_stride, const long long *slots, int n,
                                                                 int window) {
    extern __shared__ __align__(16) unsigned char store_sm[];
    T *xs = reinterpret_cast<T *>(store_sm); // [run][hd]
    __shared__ unsigned s_max[kStoreThreads / 32];
    __shared__ int s_run[kStoreThreads / 32];
    const int head = blockIdx.y, side = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int P = c.page, hd = c.hd, hdp = c.hdp;
    const T *src = side ? v : k;
    const long long stride = side ? v_stride : k_stride, most = (long long)c.n_pages << c.page_shift;
    int8_t *codes = side ? c.v : c.k;
    const int t1 = min(n, (int)(blockIdx.x + 1) * window);
    for (int t = blockIdx.x * window; t < t1; t++) {
        const long long slot = slots[t];
        if (slot < 0) continue; // skipped by the caller, or by a plan that failed
        if (slot >= most) {
            if (tid == 0) atomicOr(c.status, TQ_KV_STATUS_PAGE);
            continue;
        }
        const long long before = t ? slots[t - 1] : -1;
        const int id = (int)(slot >> c.page_shift), off = (int)slot & (P - 1);
        if (before >= 0 && (before >> c.page_shift) == id) { // not the first of its run
            if (before + 1 != slot && tid == 0) atomicOr(c.status, TQ_KV_STATUS_SLOTS);
            continue;
        }
        // the run's length: tokens t, t + 1, .. in slots slot, slot + 1, .. of this page
        const bool in = tid < P - off && tid < n - t && slots[t + tid] == slot + tid;
        const unsigned miss = ~__ballot_sync(0xffffffffu, in);
        if (lane == 0) s_run[warp] = miss ? __ffs(miss) - 1 : 32;
        __syncthreads();
        int run = s_run[0];
#pragma unroll
        for (int w = 1; w < kStoreThreads / 32; w++)
            if (run == 32 * w) run += s_run[w];
        // the run into shared memory, and its largest magnitude
        unsigned mx = 0;
        const T *base = src + (size_t)t * stride + (size_t)head * hd;
        if (VEC) {
            constexpr int E = 16 / sizeof(T);
            const int per = hd / E;
            for (int e = tid; e < run * per; e += kStoreThreads) {
                const int r = e / per, j = e - r * per;
                uint4 w = *reinterpret_cast<const uint4 *>(base + (size_t)r * stride + j * E);
                *reinterpret_cast<uint4 *>(xs + r * hd + j * E) = w;
                const T *x = reinterpret_cast<const T *>(&w);
#pragma unroll
                for (int u = 0; u < E; u++) mx = max(mx, __float_as_uint(to_f(x[u])) & 0x7fffffffu);
            }
        } else {
            for (int e = tid; e < run * hd; e += kStoreThreads) {
                const int r = e / hd, j = e - r * hd;
                const T x = base[(size_t)r * stride + j];
                xs[e] = x;
                mx = max(mx, __float_as_uint(to_f(x)) & 0x7fffffffu);
            }
        }
        mx = __reduce_max_sync(0xffffffffu, mx);
        if (lane == 0) s_max[warp] = mx;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kStoreThreads / 32; w++) mx = max(mx, s_max[w]);
        float *place = reinterpret_cast<float *>(c.scale + (size_t)id * c.n_kv + head) + side;
        float now = mx < 0x7f800000u ? __fdiv_rn(__uint_as_float(mx), 127.f) : __uint_as_float(0x7fc00000u);
        const float was = off ? *place : 0.f;
        if (off && !(now >= was)) now = now != now ? now : was; // the larger; a NaN stays
        const bool grew = off && now != was && now == now;
        const float inv = __fdiv_rn(1.f, now), ratio = __fdiv_rn(was, now);
        int8_t *page = codes + kv_block_offset(c, id, head, 0);
        const int end = off + run;
        if (side == 0) {
            const int chunks = hdp / 16;
            for (int e = tid + (grew ? 0 : off * chunks); e < end * chunks; e += kStoreThreads) {
                const int r = e / chunks, d0 = (e - r * chunks) * 16;
                if (d0 >= hd) continue; // padding: stays zero
                uint4 *dst = reinterpret_cast<uint4 *>(page + (size_t)(r >> 4) * 16 * hdp +
                                                       kv_key_offset(hdp, r & 15, d0));
                unsigned w[4] = {0, 0, 0, 0};
                if (r < off) {
                    const uint4 o = *dst;
                    const unsigned ow[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
                    for (int u = 0; u < 16; u++)
                        w[u >> 2] |= ((unsigned)recode((int)(int8_t)byte_of(ow[u >> 2], u & 3), was, now, ratio) & 0xffu)
                                     << (8 * (u & 3));
                } else {
                    const T *x = xs + (r - off) * hd + d0;
#pragma unroll
                    for (int u = 0; u < 16; u++)
                        if (d0 + u < hd) w[u >> 2] |= ((unsigned)code_of(to_f(x[u]), now, inv) & 0xffu) << (8 * (u & 3));
                }
                *dst = make_uint4(w[0], w[1], w[2], w[3]);
            }
        } else {
            const int b0 = grew ? 0 : off >> 4, nb = ((end + 15) >> 4) - b0;
            for (int e = tid; e < nb * hd; e += kStoreThreads) {
                const int b = e / hd, d = e - b * hd, r0 = (b0 + b) << 4;
                uint4 *dst = reinterpret_cast<uint4 *>(page + (size_t)(b0 + b) * 16 * hdp + d * 16);
                unsigned w[4] = {0, 0, 0, 0};
                if (r0 < off || r0 + 16 > end) {
                    const uint4 o = *dst;
                    w[0] = o.x, w[1] = o.y, w[2] = o.z, w[3] = o.w;
                }
#pragma unroll
                for (int u = 0; u < 16; u++) {
                    const int r = r0 + u, sh = 8 * (u & 3);
                    unsigned q;
                    if (r >= off && r < end)
                        q = (unsigned)code_of(to_f(xs[(r - off) * hd + d]), now, inv);
                    else if (r < off && grew)
                        q = (unsigned)recode((int)(int8_t)byte_of(w[u >> 2], u & 3), was, now, ratio);
                    else
                        continue;
                    w[u >> 2] = (w[u >> 2] & ~(0xffu << sh)) | ((q & 0xffu) << sh);
                }
                *dst = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
        __syncthreads(); // every thread has read the scale and the staged run
        if (tid == 0) *place = now;
    }
}

// ---- pages in and out --------------------------------------------------------------
// Block (listed page, head). Word e of 4 codes: keys (row r, dimensions d..d+3);
// values (block b, dimensions d..d+3, all 16 positions: four words transposed).

// b[j] = byte j of a, c, d, e in that order.
__device__ __forceinline__ void transpose4(const unsigned (&a)[4], unsigned (&b)[4]) {
    const unsigned l0 = __byte_perm(a[0], a[1], 0x5140), l1 = __byte_perm(a[2], a[3], 0x5140);
    const unsigned h0 = __byte_perm(a[0], a[1], 0x7362), h1 = __byte_perm(a[2], a[3], 0x7362);
    b[0] = __byte_perm(l0, l1, 0x5410);
    b[1] = __byte_perm(l0, l1, 0x7632);
    b[2] = __byte_perm(h0, h1, 0x5410);
    b[3] = __byte_perm(h0, h1, 0x7632);
}

__device__ __forceinline__ bool page_of(const TqKvView &c, const int *pages, int i, int *id) {
    *id = pages[i];
    if (*id >= 0 && *id < c.n_pages) return true;
    if (threadIdx.x == 0) atomicOr(c.status, TQ_KV_STATUS_PAGE);
    return false;
}

struct WriteValues {
    float *p;
    float s;
    __device__ __forceinline__ void operator()(size_t at, unsigned w) const {
        *reinterpret_cast<float4 *>(p + at) =
            make_float4((float)(int8_t)byte_of(w, 0) * s, (float)(int8_t)byte_of(w, 1) * s,
                        (float)(int8_t)byte_of(w, 2) * s, (float)(int8_t)byte_of(w, 3) * s);
    }
};
struct WriteCodes {
    int8_t *p;
    float s;
    __device__ __forceinline__ void operator()(size_t at, unsigned w) const {
        *reinterpret_cast<unsigned *>(p + at) = w;
    }
};

// Codes of a page and head to W at [row][n_kv][hd] element offsets from `to`.
template <class W>
__device__ __forceinline__ void page_out(const TqKvView &c, int id, int head, size_t to, const W &wk, const W &wv) {
    const int hd = c.hd, hdp = c.hdp, q = hd / 4, row = c.n_kv * hd;
    const int8_t *pk = c.k + kv_block_offset(c, id, head, 0), *pv = c.v + kv_block_offset(c, id, head, 0);
    for (int e = threadIdx.x; e < c.page * q; e += blockDim.x) {
        const int r = e / q, d = (e - r * q) * 4;
        const unsigned w =
            *reinterpret_cast<const unsigned *>(pk + (size_t)(r >> 4) * 16 * hdp + kv_key_offset(hdp, r & 15, d));
        wk(to + (size_t)r * row + d, w);
    }
    for (int e = threadIdx.x; e < (c.page >> 4) * q; e += blockDim.x) {
        const int b = e / q, d = (e - b * q) * 4;
        const uint4 *p = reinterpret_cast<const uint4 *>(pv + (size_t)b * 16 * hdp + d * 16);
        const uint4 x[4] = {p[0], p[1], p[2], p[3]};
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const unsigned a[4] = {(&x[0].x)[u], (&x[1].x)[u], (&x[2].x)[u], (&x[3].x)[u]};
            unsigned t[4];
            transpose4(a, t);
#pragma unroll
            for (int j = 0; j < 4; j++) wv(to + (size_t)(16 * b + 4 * u + j) * row + d, t[j]);
        }
    }
}

__global__ void kv_read_kernel(TqKvView c, const int *pages, float *k, float *v) {
    int id;
    if (!page_of(c, pages, blockIdx.x, &id)) return;
    const float2 s = c.scale[(size_t)id * c.n_kv + blockIdx.y];
    const size_t to = ((size_t)blockIdx.x * c.page * c.n_kv + blockIdx.y) * c.hd;
    page_out(c, id, blockIdx.y, to, WriteValues{k, s.x}, WriteValues{v, s.y});
}

__global__ void kv_save_kernel(TqKvView c, const int *pages, int8_t *k, int8_t *v, float *ks, float *vs) {
    int id;
    if (!page_of(c, pages, blockIdx.x, &id)) return;
    const float2 s = c.scale[(size_t)id * c.n_kv + blockIdx.y];
    const size_t to = ((size_t)blockIdx.x * c.page * c.n_kv + blockIdx.y) * c.hd;
    page_out(c, id, blockIdx.y, to, WriteCodes{k, 0.f}, WriteCodes{v, 0.f});
    if (threadIdx.x == 0) {
        ks[(size_t)blockIdx.x * c.n_kv + blockIdx.y] = s.x;
        vs[(size_t)blockIdx.x * c.n_kv + blockIdx.y] = s.y;
    }
}

// -128 is no code of the cache: -127 in its place.
__device__ __forceinline__ unsigned no_min(unsigned w) { return __vmaxs4(w, 0x81818181u); }

__global__ void kv_load_kernel(TqKvView c, const int *pages, const int8_t *k, const int8_t *v, const float *ks,
                               const float *vs) {
    int id;
    if (!page_of(c, pages, blockIdx.x, &id)) return;
    const int head = blockIdx.y, hd = c.hd, hdp = c.hdp, q = hd / 4, row = c.n_kv * hd;
    const size_t from = ((size_t)blockIdx.x * c.page * c.n_kv + head) * hd;
    int8_t *pk = c.k + kv_block_offset(c, id, head, 0), *pv = c.v + kv_block_offset(c, id, head, 0);
    for (int e = threadIdx.x; e < c.page * q; e += blockDim.x) {
        const int r = e / q, d = (e - r * q) * 4;
        const unsigned w = *reinterpret_cast<const unsigned *>(k + from + (size_t)r * row + d);
        *reinterpret_cast<unsigned *>(pk + (size_t)(r >> 4) * 16 * hdp + kv_key_offset(hdp, r & 15, d)) = no_min(w);
    }
    for (int e = threadIdx.x; e < (c.page >> 4) * q; e += blockDim.x) {
        const int b = e / q, d = (e - b * q) * 4;
        unsigned x[4][4]; // [dimension][4 positions a word]
#pragma unroll
        for (int u = 0; u < 4; u++) {
            unsigned a[4], t[4];
#pragma unroll
            for (int j = 0; j < 4; j++)
                a[j] = no_min(*reinterpret_cast<const unsigned *>(v + from + (size_t)(16 * b + 4 * u + j) * row + d));
            transpose4(a, t);
#pragma unroll
            for (int j = 0; j < 4; j++) x[j][u] = t[j];
        }
        uint4 *p = reinterpret_cast<uint4 *>(pv + (size_t)b * 16 * hdp + d * 16);
#pragma unroll
        for (int j = 0; j < 4; j++) p[j] = make_uint4(x[j][0], x[j][1], x[j][2], x[j][3]);
    }
    if (threadIdx.x == 0)
        c.scale[(size_t)id * c.n_kv + head] = make_float2(ks[(size_t)blockIdx.x * c.n_kv + head],
                                                          vs[(size_t)blockIdx.x * c.n_kv + head]);
}

constexpr int kPageThreads = 256;

template <typename T>
cudaError_t launch_store(const TqKvView &c, const T *k, const T *v, long long ks, long long vs, const long long *slots,
                         int n, cudaStream_t st) {
    const size_t smem = (size_t)c.page * c.hd * sizeof(T);
    static TqDeviceOnce once;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess)
        e = tq_device_once(once, dev, [] {
            const int most = kMaxPage * 256 * (int)sizeof(T);
            cudaError_t r =
                cudaFuncSetAttribute(kv_store_kernel<T, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
            if (r == cudaSuccess)
                r = cudaFuncSetAttribute(kv_store_kernel<T, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
            return r;
        });
    if (e != cudaSuccess) return e;
    // A decode step's tokens are runs of one: a block each. In a prompt most
    // tokens are not the first of their page, so a block looks through several.
    const int window = n <= 1024 ? 1 : TQ_KV_BLOCK;
    const dim3 grid((n + window - 1) / window, c.n_kv, 2);
    const size_t ax = (uintptr_t)k | (uintptr_t)v | (size_t)(ks * (long long)sizeof(T)) |
                      (size_t)(vs * (long long)sizeof(T)) | (size_t)c.hd * sizeof(T);
    if (ax % 16 == 0)
        kv_store_kernel<T, true><<<grid, kStoreThreads, smem, st>>>(c, k, v, ks, vs, slots, n, window);
    else
        kv_store_kernel<T, false><<<grid, kStoreThreads, smem, st>>>(c, k, v, ks, vs, slots, n, window);
    return cudaGetLastError();
}

} // namespace

cudaError_t tq_kv_launch_store(const TqKvView &v, const void *k, const void *val, int dtype, long long k_stride,
                               long long v_stride, const long long *slots, int n, cudaStream_t st) {
    if (n == 0) return cudaSuccess;
    if (dtype == TQ_LINEAR_F32)
        return launch_store(v, (const float *)k, (const float *)val, k_stride, v_stride, slots, n, st);
    if (dtype == TQ_LINEAR_F16)
        return launch_store(v, (const __half *)k, (const __half *)val, k_stride, v_stride, slots, n, st);
    return launch_store(v, (const __nv_bfloat16 *)k, (const __nv_bfloat16 *)val, k_stride, v_stride, slots, n, st);
}

cudaError_t tq_kv_launch_load(const TqKvView &v, const int *pages, int n, const int8_t *k, const int8_t *val,
                              const float *kscale, const float *vscale, cudaStream_t st) {
    if (n == 0) return cudaSuccess;
    kv_load_kernel<<<dim3(n, v.n_kv), kPageThreads, 0, st>>>(v, pages, k, val, kscale, vscale);
    return cudaGetLastError();
}

cudaError_t tq_kv_launch_save(const TqKvView &v, const int *pages, int n, int8_t *k, int8_t *val, float *kscale,
                              float *vscale, cudaStream_t st) {
    if (n == 0) return cudaSuccess;
    kv_save_kernel<<<dim3(n, v.n_kv), kPageThreads, 0, st>>>(v, pages, k, val, kscale, vscale);
    return cudaGetLastError();
}

cudaError_t tq_kv_launch_read(const TqKvView &v, const int *pages, int n, float *k, float *val, cudaStream_t st) {
    if (n == 0) return cudaSuccess;
    kv_read_kernel<<<dim3(n, v.n_kv), kPageThreads, 0, st>>>(v, pages, k, val);
    return cudaGetLastError();
}
