// tq_kv_attn.cuh — what the two attention kernels over the paged 8-bit cache
// share (tq_kv_attn.cu: few rows; tq_kv_prompt.cu: many).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "tq_common.cuh"
#include "tq_kv.h"
#include "tq_ptx.cuh"

struct TqKvParams {
    TqKvView c;
    TqKvAttn a;
    int group, vec, shift_sums; // prefix entry = 2^shift_sums sequences
    int tokens_cut;             // sequences of more new tokens are the prompt kernel's
    float scale2;               // scale * log2(e)
};
constexpr int kKvSums = 512;                      // entries of the prefix sums
constexpr size_t kKvHead = TQ_KV_WORKSPACE_HEAD; // workspace: arrival counters first

namespace tqkv {

struct Seq { // what a sequence's lengths say
    int start, nq, len;
};

__device__ __forceinline__ void cvt4(unsigned u, unsigned &lo, unsigned &hi) {
    // codes + 128 under the exponent of 1024, then minus 1152: exact
    const unsigned a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 off = __half2half2(__ushort_as_half(0x6480));
    const __half2 x = __hsub2(*reinterpret_cast<const __half2 *>(&a), off);
    const __half2 y = __hsub2(*reinterpret_cast<const __half2 *>(&b), off);
    lo = *reinterpret_cast<const unsigned *>(&x);
    hi = *reinterpret_cast<const unsigned *>(&y);
}
__device__ __forceinline__ unsigned pack2(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const unsigned *>(&h);
}
__device__ __forceinline__ float2 unpack2(unsigned u) { return __half22float2(*reinterpret_cast<const __half2 *>(&u)); }

// 2^x to about 2^-22 of it; below 2^-126 it is 0, which no sum here can tell.
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kLeast = 1e-30f; // least score factor of a block: -inf times it stays -inf
constexpr float kFar = 0x1p20f;  // scores (in powers of two) from which on a weight could leave float16 by their rounding
constexpr float kLeastValue = 0x1p-92f; // value scales below count as 0: the sums that hold their inverse stay finite
constexpr float kNoValue = 0x1p-60f;    // what such a scale, of no values, counts as beside others

__device__ __forceinline__ void mma16816(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T> struct Elem;
template <> struct Elem<float> {
    static __device__ __forceinline__ float get(const float *p) { return *p; }
    static __device__ __forceinline__ void put2(float *p, float x, float y, bool vec) {
        if (vec)
            *reinterpret_cast<float2 *>(p) = make_float2(x, y);
        else {
            p[0] = x;
            p[1] = y;
        }
    }
};
template <> struct Elem<__half> {
    static __device__ __forceinline__ float get(const __half *p) { return __half2float(*p); }
    static __device__ __forceinline__ void put2(__half *p, float x, float y, bool vec) {
        if (vec)
            *reinterpret_cast<__half2 *>(p) = __floats2half2_rn(x, y);
        else {
            p[0] = __float2half_rn(x);
            p[1] = __float2half_rn(y);
        }
    }
};
template <> struct Elem<__nv_bfloat16> {
    static __device__ __forceinline__ float get(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
    static __device__ __forceinline__ void put2(__nv_bfloat16 *p, float x, float y, bool vec) {
        if (vec)
            *reinterpret_cast<__nv_bfloat162 *>(p) = __floats2bfloat162_rn(x, y);
        else {
            p[0] = __float2bfloat16_rn(x);
            p[1] = __float2bfloat16_rn(y);
        }
    }
};

// A sequence's lengths, checked: one that cannot be served has no tokens.
__device__ __forceinline__ Seq seq_at(const TqKvParams &p, const int *starts, const int *lens, int i) {
    Seq s;
    s.start = starts[i];
    const int e = starts[i + 1];
    s.nq = e - s.start;
    s.len = lens[i];
    if (s.start < 0 || e < s.start || e > p.a.n_tokens || s.len < 0) {
        s.nq = s.len = 0;
        atomicOr(p.c.status, TQ_KV_STATUS_LENGTH);
    }
    if (s.len > p.a.table_cols << p.c.page_shift) {
        s.nq = s.len = 0;
        atomicOr(p.c.status, TQ_KV_STATUS_TABLE);
    }
    return s;
}

// Bounded wait for an mbarrier. What it waits for always arrives; should it not, the status says so and no later wait of the CTA waits.
__device__ __forceinline__ void wait_long(uint64_t *bar, unsigned parity, volatile int *late, unsigned *status) {
    unsigned long long t0 = 0;
    for (unsigned it = 1; !*late; it++) {
        if (tqp::mbar_try_wait_hint(bar, parity, 200000u)) return;
        if (it % 64 == 0) { // reading the clock costs more than most waits last
            const unsigned long long now = tqp::global_ns();
            if (t0 == 0) t0 = now;
            if (now - t0 > tqp::kWaitNs) {
                atomicOr(status, TQ_KV_STATUS_TIMEOUT);
                *late = 1;
            }
        }
    }
}
__device__ __forceinline__ void wait_slot(uint64_t *bar, unsigned parity, volatile int *late, unsigned *status) {
    if (!tqp::mbar_try_wait(bar, parity)) wait_long(bar, parity, late, status);
}

// The power of two that brings a row's largest magnitude to 2^13 .. 2^14: float16
// pieces keep their bits far below it (magnitudes under 2^-87 count as 2^-87).
// *back: its inverse.
__device__ __forceinline__ float row_scale(float big, float *back) {
    const int e = max(40, (int)(__float_as_uint(big) >> 23)); // its exponent + 127; 255 for an infinity
    *back = __uint_as_float((unsigned)(e - 13) << 23);
    return __uint_as_float((unsigned)(267 - e) << 23);
}

} // namespace tqkv

// Many rows a sequence on the tensor cores; hdp 64 or 128 (tq_kv_prompt.cu).
size_t tq_kv_prompt_workspace(int hdp, int sms);
cudaError_t tq_kv_launch_prompt(const TqKvParams &p, int sms, cudaStream_t st);
