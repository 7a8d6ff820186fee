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
// The run is read once, 16 bytes a thread, and stays in shared memory in its own
// type, because the codes need the maximum first; a value block is written two
// dimensions a thread, each one 16-byte word.
//
// Bound. One token a sequence: latency, 3.8 us for 32 sequences of 4 heads of 128
// (the slot, the tokens and the scale), 4.4 with the pages in 24 caches in turn,
// 8.3 there if every page's scale grows: its held codes are read, rounded again and
// written. (A decode step's pages seldom grow: the largest of a page's positions
// sets its scale.) A prompt:
// 7,096 bfloat16 tokens of 4 heads of 128 take 21 us for 22 MB, half of it issue
// slots (a code is about 6 instructions), the rest waiting at the two barriers of
// a block with 1.3 waves of blocks; 16,000 tokens of 8 float32 heads of 128, 164 MB,
// take 61 us, 2.7 TB/s (41% of the measured copy).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "tq_common.cuh"
#include "tq_kv.h"

namespace {

constexpr int kStoreThreads = 1024; // at most; 128 for little pages
constexpr int kStoreWarps = kStoreThreads / 32;
constexpr int kMaxPage = 128, kLeastThreads = 128;
constexpr int kFewTokens = 128; // up to these, runs of one (a decode step) are likelier than a prompt
static_assert(kLeastThreads >= kMaxPage, "one thread per token of a run");
constexpr float kRound = 12582912.f; // 1.5 * 2^23: x + kRound holds the integer nearest to x in its low bits

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }

// The integer nearest to x / s (ties to even), |x| <= 127 s up to rounding.
__device__ __noinline__ unsigned code_exact(float x, float s, float inv) {
    if (!(s > 0.f)) return 0; // zero or NaN
    if (s < 0x1p-100f)        // the products below could underflow
        return (unsigned)(int)fmin(fmax(rint(__ddiv_rn((double)x, (double)s)), -127.0), 127.0);
    const float y = __fmul_rn(x, inv), lo = floorf(y);
    float t = rintf(y);
    if (fabsf(y - t) > 0.4999f) { // the half between lo and lo + 1 decides
        const float r = __fmaf_rn(-(lo + 0.5f), s, x);
        t = r > 0.f ? lo + 1.f : r < 0.f ? lo : 2.f * rintf(0.5f * (lo + 0.5f));
    }
    return (unsigned)(int)fminf(fmaxf(t, -127.f), 127.f);
}

// Four codes, a byte each. easy: the scale is neither zero, NaN nor tiny.
__device__ __forceinline__ unsigned codes4(const float (&x)[4], float s, float inv, bool easy) {
    float v[4], off = easy ? 0.f : 1.f;
#pragma unroll
    for (int u = 0; u < 4; u++) {
        const float y = __fmul_rn(x[u], inv);
        v[u] = __fadd_rn(y, kRound);
        off = fmaxf(off, fabsf(__fadd_rn(y, -__fadd_rn(v[u], -kRound)))); // from the nearest integer
    }
    if (off > 0.4999f) // rare: next to a half
        return (code_exact(x[0], s, inv) & 0xffu) | (code_exact(x[1], s, inv) & 0xffu) << 8 |
               (code_exact(x[2], s, inv) & 0xffu) << 16 | code_exact(x[3], s, inv) << 24;
    return __byte_perm(__byte_perm(__float_as_uint(v[0]), __float_as_uint(v[1]), 0x0040),
                       __byte_perm(__float_as_uint(v[2]), __float_as_uint(v[3]), 0x0040), 0x5410);
}

// The integer nearest to c * was / now (ties to even).
__device__ __forceinline__ unsigned recode(unsigned byte, float was, float now, float ratio) {
    const float c = (float)(int8_t)byte, y = __fmul_rn(c, ratio), v = __fadd_rn(y, kRound);
    if (fabsf(__fadd_rn(y, -__fadd_rn(v, -kRound))) > 0.4999f)
        return (unsigned)(int)rint(__ddiv_rn((double)c * (double)was, (double)now)) & 0xffu;
    return __float_as_uint(v) & 0xffu;
}
__device__ __noinline__ unsigned recode4(unsigned held, float was, float now, float ratio) { // four held codes
    const unsigned w = held ^ TQ_KV_BIAS;
    return (recode(w & 0xffu, was, now, ratio) | recode(w >> 8 & 0xffu, was, now, ratio) << 8 |
            recode(w >> 16 & 0xffu, was, now, ratio) << 16 | recode(w >> 24, was, now, ratio) << 24) ^
           TQ_KV_BIAS;
}

// e / per and e % per for e = threadIdx.x, + blockDim.x, ..: one division, then steps.
struct Places {
    int q, r, dq, dr, per;
    __device__ __forceinline__ explicit Places(int n) : per(n) {
        q = threadIdx.x / per, r = threadIdx.x - q * per;
        dq = blockDim.x / per, dr = blockDim.x - dq * per;
    }
    __device__ __forceinline__ void step() {
        q += dq, r += dr;
        if (r >= per) r -= per, q++;
    }
};

// Two neighbouring elements, widened.
__device__ __forceinline__ float2 pair_at(const float *p) { return *reinterpret_cast<const float2 *>(p); }
__device__ __forceinline__ float2 pair_at(const __half *p) { return __half22float2(*reinterpret_cast<const __half2 *>(p)); }
__device__ __forceinline__ float2 pair_at(const __nv_bfloat16 *p) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(p));
}
// Eight, 16-byte aligned.
template <typename T> __device__ __forceinline__ void eight_at(const T *p, float (&x)[8]) {
    constexpr int E = 16 / sizeof(T);
#pragma unroll
    for (int j = 0; j < 8 / E; j++) {
        const uint4 w = *reinterpret_cast<const uint4 *>(p + j * E);
#pragma unroll
        for (int u = 0; u < E; u++) x[j * E + u] = to_f(reinterpret_cast<const T *>(&w)[u]);
    }
}

__device__ __forceinline__ unsigned byte_of(unsigned w, int i) { return (w >> (8 * i)) & 0xffu; }

template <typename T, bool VEC>
__global__ void __launch_bounds__(kStoreThreads, 1) kv_store_kernel(TqKvView c, const T *k, const T *v, long long k_stride,
                                                                 long long v_stride, const long long *slots, int n,
                                                                 int window) {
    extern __shared__ __align__(16) unsigned char store_sm[];
    T *xs = reinterpret_cast<T *>(store_sm); // [run][hd]
    __shared__ unsigned s_max[kStoreWarps];
    __shared__ int s_run[kStoreWarps];
    const int head = blockIdx.y, side = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int P = c.page, hd = c.hd, hdp = c.hdp;
    const T *src = side ? v : k;
    const long long stride = side ? v_stride : k_stride, most = (long long)c.n_pages << c.page_shift;
    int8_t *codes = side ? c.v : c.k;
    // the tokens of this window that begin a run: a lane each, in every warp
    const int t0 = blockIdx.x * window, mine = t0 + lane;
    unsigned firsts;
    const long long lane_slot = lane < window && mine < n ? slots[mine] : -1;
    {
        const long long slot = lane_slot, before = lane < window && mine < n && mine ? slots[mine - 1] : -1;
        const bool there = slot >= 0 && slot < most; // negative: skipped by the caller, or by a plan that failed
        const bool goes_on = there && before >= 0 && (before >> c.page_shift) == (slot >> c.page_shift);
        if (warp == 0 && slot >= most) atomicOr(c.status, TQ_KV_STATUS_PAGE);
        if (warp == 0 && goes_on && before + 1 != slot) atomicOr(c.status, TQ_KV_STATUS_SLOTS);
        firsts = __ballot_sync(0xffffffffu, there && !goes_on);
    }
    for (; firsts; firsts &= firsts - 1) {
        const int t = t0 + __ffs(firsts) - 1;
        const long long slot = __shfl_sync(0xffffffffu, lane_slot, t - t0);
        const int id = (int)(slot >> c.page_shift), off = (int)slot & (P - 1);
        float *place = reinterpret_cast<float *>(c.scale + (size_t)id * c.n_kv + head) + side;
        const float held = off ? *place : 0.f;
        // the run's length: tokens t, t + 1, .. in slots slot, slot + 1, .. of this page
        const bool in = tid < P - off && tid < n - t && slots[t + tid] == slot + tid;
        const unsigned miss = ~__ballot_sync(0xffffffffu, in);
        if (lane == 0) s_run[warp] = miss ? __ffs(miss) - 1 : 32;
        __syncthreads();
        int run = s_run[0];
#pragma unroll
        for (int w = 1; w < kMaxPage / 32; w++)
            if (run == 32 * w) run += s_run[w];
        // the run into shared memory, and its largest magnitude
        unsigned mx = 0;
        const T *base = src + (size_t)t * stride + (size_t)head * hd;
        if (VEC) {
            constexpr int E = 16 / sizeof(T);
            Places at(hd / E);
#pragma unroll 4
            for (int e = tid; e < run * at.per; e += blockDim.x, at.step()) {
                const uint4 w = *reinterpret_cast<const uint4 *>(base + (size_t)at.q * stride + at.r * E);
                *reinterpret_cast<uint4 *>(xs + e * E) = w;
                const T *x = reinterpret_cast<const T *>(&w);
#pragma unroll
                for (int u = 0; u < E; u++) mx = max(mx, __float_as_uint(to_f(x[u])) & 0x7fffffffu);
            }
        } else {
            Places at(hd);
            for (int e = tid; e < run * hd; e += blockDim.x, at.step()) {
                const T x = base[(size_t)at.q * stride + at.r];
                xs[e] = x;
                mx = max(mx, __float_as_uint(to_f(x)) & 0x7fffffffu);
            }
        }
        mx = __reduce_max_sync(0xffffffffu, mx);
        if (lane == 0) s_max[warp] = mx;
        __syncthreads();
        mx = __reduce_max_sync(0xffffffffu, lane < (int)blockDim.x >> 5 ? s_max[lane] : 0u);
        float now = mx < 0x7f800000u ? __fdiv_rn(__uint_as_float(mx), 127.f) : __uint_as_float(0x7fc00000u);
        const float was = held;
        if (off && !(now >= was)) now = now != now ? now : was; // the larger; a NaN stays
        const bool grew = off && now != was && now == now, easy = now >= 0x1p-100f;
        const float inv = __fdiv_rn(1.f, now), ratio = __fdiv_rn(was, now);
        int8_t *page = codes + kv_block_offset(c, id, head, 0);
        const int end = off + run;
        if (side == 0) {
            const int chunks = hdp / 16, shift = __ffs(chunks) - 1;
            for (int e = tid + (grew ? 0 : off << shift); e < end << shift; e += blockDim.x) {
                const int r = e >> shift, d0 = (e - (r << shift)) * 16;
                if (d0 >= hd) continue; // padding: keeps code 0
                uint4 *dst = reinterpret_cast<uint4 *>(page + (size_t)(r >> 4) * 16 * hdp +
                                                       kv_key_offset(hdp, r & 15, d0));
                uint4 w;
                if (r < off) {
                    const uint4 o = *dst;
                    w = make_uint4(recode4(o.x, was, now, ratio), recode4(o.y, was, now, ratio),
                                   recode4(o.z, was, now, ratio), recode4(o.w, was, now, ratio));
                } else {
                    const T *x = xs + (r - off) * hd + d0;
#pragma unroll
                    for (int q = 0; q < 4; q += 2) {
                        float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                        if (d0 + 4 * q < hd) eight_at(x + 4 * q, y);
                        (&w.x)[q] = codes4({y[0], y[1], y[2], y[3]}, now, inv, easy) ^ TQ_KV_BIAS;
                        (&w.x)[q + 1] = codes4({y[4], y[5], y[6], y[7]}, now, inv, easy) ^ TQ_KV_BIAS;
                    }
                }
                *dst = w;
            }
        } else {
            // a thread: two dimensions of a block, so that a token's pair is one read
            const int b0 = grew ? 0 : off >> 4, nb = ((end + 15) >> 4) - b0;
            Places at(hd / 2);
            for (int e = tid; e < nb * (hd / 2); e += blockDim.x, at.step()) {
                const int d = 2 * at.r, r0 = (b0 + at.q) << 4;
                uint4 *dst = reinterpret_cast<uint4 *>(page + (size_t)(b0 + at.q) * 16 * hdp + d * 16);
                uint4 w[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
                const bool all = r0 >= off && r0 + 16 <= end; // else some positions stay, or are rounded again
                if (!all) w[0] = dst[0], w[1] = dst[1];
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const int r = r0 + 4 * q - off; // first of four tokens, in the run
                    if (!all && grew && r < 0) { // positions before the run
                        const unsigned old = r + 3 < 0 ? 0xffffffffu : 0xffffffffu >> 8 * (r + 4);
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            unsigned &o = (&w[h].x)[q];
                            o = (o & ~old) | (recode4(o, was, now, ratio) & old);
                        }
                    }
                    if (!all && (r + 3 < 0 || r >= run)) continue;
                    float y[2][4];
                    unsigned keep = 0;
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        const bool fresh = all || (r + u >= 0 && r + u < run);
                        const float2 z = fresh ? pair_at(xs + (r + u) * hd + d) : make_float2(0.f, 0.f);
                        y[0][u] = z.x, y[1][u] = z.y;
                        if (!fresh) keep |= 0xffu << 8 * u;
                    }
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        unsigned &o = (&w[h].x)[q];
                        o = (o & keep) | ((codes4(y[h], now, inv, easy) ^ TQ_KV_BIAS) & ~keep);
                    }
                }
                dst[0] = w[0], dst[1] = w[1];
            }
        }
        if (tid == 0) *place = now;
        __syncthreads(); // the staged run is read
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

// Codes of a page and head to W at [row][n_kv][hd] element offsets from `to`; keys (side 0) or values.
template <class W>
__device__ __forceinline__ void page_out(const TqKvView &c, int id, int head, size_t to, const W &wk, const W &wv,
                                         int side) {
    const int hd = c.hd, hdp = c.hdp, q = hd / 4, row = c.n_kv * hd;
    const int8_t *pk = c.k + kv_block_offset(c, id, head, 0), *pv = c.v + kv_block_offset(c, id, head, 0);
#pragma unroll 4
    for (int e = threadIdx.x; side == 0 && e < c.page * q; e += blockDim.x) {
        const int r = e / q, d = (e - r * q) * 4;
        const unsigned w =
            *reinterpret_cast<const unsigned *>(pk + (size_t)(r >> 4) * 16 * hdp + kv_key_offset(hdp, r & 15, d));
        wk(to + (size_t)r * row + d, w ^ TQ_KV_BIAS);
    }
    for (int e = threadIdx.x; side == 1 && e < (c.page >> 4) * q; e += blockDim.x) {
        const int b = e / q, d = (e - b * q) * 4;
        const uint4 *p = reinterpret_cast<const uint4 *>(pv + (size_t)b * 16 * hdp + d * 16);
        const uint4 x[4] = {p[0], p[1], p[2], p[3]};
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const unsigned a[4] = {(&x[0].x)[u], (&x[1].x)[u], (&x[2].x)[u], (&x[3].x)[u]};
            unsigned t[4];
            transpose4(a, t);
#pragma unroll
            for (int j = 0; j < 4; j++) wv(to + (size_t)(16 * b + 4 * u + j) * row + d, t[j] ^ TQ_KV_BIAS);
        }
    }
}

__global__ void kv_read_kernel(TqKvView c, const int *pages, float *k, float *v) {
    int id;
    if (!page_of(c, pages, blockIdx.x, &id)) return;
    const float2 s = c.scale[(size_t)id * c.n_kv + blockIdx.y];
    const size_t to = ((size_t)blockIdx.x * c.page * c.n_kv + blockIdx.y) * c.hd;
    page_out(c, id, blockIdx.y, to, WriteValues{k, s.x}, WriteValues{v, s.y}, blockIdx.z);
}

__global__ void kv_save_kernel(TqKvView c, const int *pages, int8_t *k, int8_t *v, float *ks, float *vs) {
    int id;
    if (!page_of(c, pages, blockIdx.x, &id)) return;
    const float2 s = c.scale[(size_t)id * c.n_kv + blockIdx.y];
    const size_t to = ((size_t)blockIdx.x * c.page * c.n_kv + blockIdx.y) * c.hd;
    page_out(c, id, blockIdx.y, to, WriteCodes{k, 0.f}, WriteCodes{v, 0.f}, blockIdx.z);
    if (threadIdx.x == 0 && blockIdx.z == 0) {
        ks[(size_t)blockIdx.x * c.n_kv + blockIdx.y] = s.x;
        vs[(size_t)blockIdx.x * c.n_kv + blockIdx.y] = s.y;
    }
}

// Four int8 codes as they are held. -128 is no code of the cache: -127 in its place.
__device__ __forceinline__ unsigned held4(unsigned w) { return __vmaxs4(w, 0x81818181u) ^ TQ_KV_BIAS; }

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
        *reinterpret_cast<unsigned *>(pk + (size_t)(r >> 4) * 16 * hdp + kv_key_offset(hdp, r & 15, d)) = held4(w);
    }
    for (int e = threadIdx.x; e < (c.page >> 4) * q; e += blockDim.x) {
        const int b = e / q, d = (e - b * q) * 4;
        unsigned x[4][4]; // [dimension][4 positions a word]
#pragma unroll
        for (int u = 0; u < 4; u++) {
            unsigned a[4], t[4];
#pragma unroll
            for (int j = 0; j < 4; j++)
                a[j] = held4(*reinterpret_cast<const unsigned *>(v + from + (size_t)(16 * b + 4 * u + j) * row + d));
            transpose4(a, t);
#pragma unroll
            for (int j = 0; j < 4; j++) x[j][u] = t[j];
        }
        uint4 *p = reinterpret_cast<uint4 *>(pv + (size_t)b * 16 * hdp + d * 16);
#pragma unroll
        for (int j = 0; j < 4; j++) p[j] = make_uint4(x[j][0], x[j][1], x[j][2], x[j][3]);
    }
    if (threadIdx.x == 0) { // a scale is a magnitude: a negative or infinite one counts as NaN
        const float a = ks[(size_t)blockIdx.x * c.n_kv + head], b = vs[(size_t)blockIdx.x * c.n_kv + head];
        const float nan = __uint_as_float(0x7fc00000u), inf = __uint_as_float(0x7f800000u);
        c.scale[(size_t)id * c.n_kv + head] = make_float2(a >= 0.f && a < inf ? a : nan, b >= 0.f && b < inf ? b : nan);
    }
}

constexpr int kPageThreads = 256;

template <typename T>
cudaError_t launch_store(const TqKvView &c, const T *k, const T *v, long long ks, long long vs, const long long *slots,
                         int n, int sms, cudaStream_t st) {
    const int rows = c.page < n ? c.page : n; // of a run, at most
    const size_t smem = (size_t)rows * c.hd * sizeof(T);
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
    const long long lines = 2ll * c.n_kv; // (head, side) pairs
    // Tokens per block, which looks for those that begin a run: a power of two, so that a prompt's
    // pages fall to the blocks evenly, for a few waves of blocks. (One token a block up to 1024:
    // 1000 tokens in a row, 8 heads of 128, bfloat16, pages of 64 took 25.7 us, now 13.1; 300
    // runs of one 12.3, now 20 to 22.)
    int window = 1;
    while (window < (c.page >= 32 ? 32 : 16) && window * 16ll * sms < n * lines) window *= 2;
    // Threads: 32 elements each of a full page, but 128 for few tokens (100 runs of one, 8 float32
    // heads of 128: 6.0 us, with 256 threads 8.9; 100 in a row 10.0 and 6.9), and no more than the
    // blocks at work (their runs fill shared memory) leave room for. One block an SM: 16000
    // tokens of 8 float32 heads of 256, pages of 128, 340 us with 256 threads and 171 with 1024.
    // Three or more: 16000 tokens of 8 bfloat16 heads of 256, 128 us with 256 and 152 with 1024.
    const long long pages = min(((long long)n / c.page + 1) * lines, (long long)sms * (228 * 1024 / (smem + 2048)));
    int threads = kLeastThreads;
    while (threads < kStoreThreads && threads * 32 < rows * c.hd && (threads < 256 ? n > kFewTokens : pages * threads < 768ll * sms))
        threads *= 2;
    const dim3 grid((n + window - 1) / window, c.n_kv, 2);
    const size_t ax = (uintptr_t)k | (uintptr_t)v | (size_t)(ks * (long long)sizeof(T)) |
                      (size_t)(vs * (long long)sizeof(T)) | (size_t)c.hd * sizeof(T);
    if (ax % 16 == 0)
        kv_store_kernel<T, true><<<grid, threads, smem, st>>>(c, k, v, ks, vs, slots, n, window);
    else
        kv_store_kernel<T, false><<<grid, threads, smem, st>>>(c, k, v, ks, vs, slots, n, window);
    return cudaGetLastError();
}

} // namespace

cudaError_t tq_kv_launch_store(const TqKvView &v, const void *k, const void *val, int dtype, long long k_stride,
                               long long v_stride, const long long *slots, int n, int sms, cudaStream_t st) {
    if (n == 0) return cudaSuccess;
    if (dtype == TQ_LINEAR_F32)
        return launch_store(v, (const float *)k, (const float *)val, k_stride, v_stride, slots, n, sms, st);
    if (dtype == TQ_LINEAR_F16)
        return launch_store(v, (const __half *)k, (const __half *)val, k_stride, v_stride, slots, n, sms, st);
    return launch_store(v, (const __nv_bfloat16 *)k, (const __nv_bfloat16 *)val, k_stride, v_stride, slots, n, sms, st);
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
    kv_save_kernel<<<dim3(n, v.n_kv, 2), kPageThreads, 0, st>>>(v, pages, k, val, kscale, vscale);
    return cudaGetLastError();
}

cudaError_t tq_kv_launch_read(const TqKvView &v, const int *pages, int n, float *k, float *val, cudaStream_t st) {
    if (n == 0) return cudaSuccess;
    kv_read_kernel<<<dim3(n, v.n_kv, 2), kPageThreads, 0, st>>>(v, pages, k, val);
    return cudaGetLastError();
}
