// tq_kv.h — the paged 8-bit key/value cache: its device layout and the
// launchers behind the tq_kv_* entry points (not part of the public ABI).
//
// A page holds `page` consecutive positions of one sequence. For each layer,
// page and KV head it holds page x hdp key codes, page x hdp value codes and
// one float32 scale for each of the two; a value is code * scale, codes are
// integers in [-127, 127], held as the byte code + 128: under the exponent of 1024
// it is a float16 but for a subtraction. hdp is the head size rounded up to 64, 128
// or 256; the padding holds zero codes. Pages are cut into blocks of 16 positions:
//   keys    block = [16 positions][hdp] bytes; the 16-byte chunk c of a row sits
//           at chunk c ^ ((row & 1) << 2) when hdp >= 128, so that eight lanes
//           reading four chunks of two adjacent rows hit distinct banks after a
//           verbatim copy into shared memory;
//   values  block = [hdp][16 positions] bytes: the 16 positions of one dimension
//           are one 16-byte word, the order in which the product p . v reads
//           them (its sum runs over positions).
// Both are 16 * hdp bytes, contiguous, and page-major:
//   code offset = ((page * n_kv + head) * page_tokens + 16 * block) * hdp.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/tensai_cuda.h"

#define TQ_KV_BLOCK 16 // positions per block
#define TQ_KV_ZERO 0x80  // the byte of code 0; a word of four int8 codes ^ TQ_KV_BIAS is what is held, and back
#define TQ_KV_BIAS 0x80808080u

struct TqKvLayer {
    int8_t *k, *v;
    float2 *scale; // [n_pages][n_kv]: key scale, value scale
};

// One layer as the kernels see it.
struct TqKvView {
    int8_t *k, *v;
    float2 *scale;
    unsigned *status; // TQ_KV_STATUS_* bits
    int n_kv, hd, hdp, page, page_shift, n_pages;
};

#ifdef __CUDACC__
// Byte of key code (position row r of a block, dimension d).
__device__ __forceinline__ int kv_key_offset(int hdp, int r, int d) {
    const int c = d >> 4;
    return r * hdp + ((hdp >= 128 ? c ^ ((r & 1) << 2) : c) << 4) + (d & 15);
}
// Start of block b of (page id, head).
__device__ __forceinline__ size_t kv_block_offset(const TqKvView &v, int id, int head, int b) {
    return ((((size_t)id * v.n_kv + head) << v.page_shift) + ((size_t)b << 4)) * v.hdp;
}
#endif

// Element types of keys, values, queries and outputs: TQ_LINEAR_F32 / F16 / BF16.
cudaError_t tq_kv_launch_plan(int page_shift, int n_pages, unsigned *status, const tq_kv_plan_args &a, cudaStream_t st);
cudaError_t tq_kv_launch_release(int page_shift, int n_pages, unsigned *status, const tq_kv_release_args &a,
                                 cudaStream_t st);
// *bits = *status, and *status = 0, in one step: what other threads' kernels report meanwhile stays.
cudaError_t tq_kv_launch_take(unsigned *status, unsigned *bits, cudaStream_t st);
cudaError_t tq_kv_launch_store(const TqKvView &v, const void *k, const void *val, int dtype, long long k_stride,
                               long long v_stride, const long long *slots, int n, int sms, cudaStream_t st);
// Plain [n][page][n_kv][hd] codes and [n][n_kv] scales <-> the listed pages.
cudaError_t tq_kv_launch_load(const TqKvView &v, const int *pages, int n, const int8_t *k, const int8_t *val,
                              const float *kscale, const float *vscale, cudaStream_t st);
cudaError_t tq_kv_launch_save(const TqKvView &v, const int *pages, int n, int8_t *k, int8_t *val, float *kscale,
                              float *vscale, cudaStream_t st);
// The values (code * scale) of the listed pages, float32.
cudaError_t tq_kv_launch_read(const TqKvView &v, const int *pages, int n, float *k, float *val, cudaStream_t st);

struct TqKvAttn {
    const void *q;
    void *out;
    int dtype;
    long long q_stride, out_stride; // elements between tokens
    int n_q, n_tokens, n;
    const int *starts, *lens, *table;
    int table_stride, table_cols;
    float scale;
    void *workspace; // zero before the first use, left zero where it has to be
};
size_t tq_kv_attn_workspace(int hdp, int sms);
cudaError_t tq_kv_launch_attn(const TqKvView &v, const TqKvAttn &a, int sms, cudaStream_t st);
