// tq_kv_prompt.cu — attention of many query rows over the paged 8-bit cache on
// the 5th-generation tensor cores (the formulas are in tq_kv_attn.cu; head sizes
// up to 128; sequences of more than rows_cut rows).
//
// The rows of a sequence and KV head (new tokens x query heads of the group) are
// cut into blocks of 256, two tiles A and B of 128 rows, positions into tiles of
// 128. For each position tile and row tile:
//   S = Q K^T    tcgen05.mma kind::f16, operands in shared memory, S in TMEM;
//   softmax      one thread a row: S from TMEM, P back over S as float16;
//   O += P V     tcgen05.mma with P from TMEM, O in TMEM.
// While the softmax of one row tile runs, the tensor cores work for the other.
// Codes become float16 once per CTA and position tile (exact), in four warps
// that go through registers: HBM/L2 -> codes -> float16 -> swizzled operand.
// Float32 queries take two float16 pieces of q and of p (22 bits): twice the
// products. 16-bit queries take one.
//
// The scales. With a_b, c_b the key and value scale of a 16-position block,
//   w_t = s_t a_b + log2 c_b,  M >= max w_t - 4 (raised only when w exceeds M + 4),
//   P = 2^(w_t - M + 10),  O = sum P v codes,  L = sum_b (sum P) / c_b,
//   out = O / L:
// the value scale rides in the exponent at no cost, and P stays below 2^14. A
// block of value scale 0 counts with c = 1 and zero codes.
//
// Work: (sequence, KV head, row block) segments x position tiles, laid end to end
// and cut evenly over one CTA per SM. A cut segment's parts go to the workspace;
// the second kernel joins them in order (a fixed order: the same bits each time).
//
// Bound by the exponentials (16 a cycle and SM) and the tensor cores alike: 128
// positions of 128 rows take about 1024 cycles of each at head size 128.
#include <climits>

#include "tq_kv_attn.cuh"

namespace {

using namespace tqkv;
using Params = TqKvParams;

constexpr int kRows = 128;      // rows of a tile
constexpr int kBlockRows = 256; // rows of a block: tiles A and B
constexpr int kPos = 128;       // positions of a tile
constexpr int kBlocks = kPos / TQ_KV_BLOCK;
constexpr int kSoftWarps = 8, kConvWarps = 4;
constexpr int kConvThreads = 32 * kConvWarps;
constexpr int kMmaWarp = kSoftWarps + kConvWarps; // one thread of it issues
constexpr int kThreads = 32 * (kMmaWarp + 1);
constexpr int kConsts = 4;      // position tiles whose scales are kept
constexpr int kMinTiles = 2;    // position tiles per CTA below which fewer CTAs work
constexpr float kSlack = 4.f;   // log2 by which w may exceed M
constexpr float kUnit = 10.f;   // log2 of P at w = M
constexpr int kJoinThreads = 256, kJoinRows = 32;

constexpr int stages_of(int hdp, int pieces) { return hdp == 128 && pieces == 2 ? 1 : 2; }
constexpr size_t operand_bytes(int hdp) { return (size_t)kPos * hdp * 2; } // a K or V tile, or a piece of a Q tile
constexpr size_t smem_bytes(int hdp, int pieces) {
    return 1024 + operand_bytes(hdp) * (2 * pieces + 2 * stages_of(hdp, pieces)) + sizeof(long long) * (kKvSums + 1);
}
constexpr size_t partial_floats(int hdp) { return (size_t)kBlockRows * (hdp + 2); }

// ---- the list of work ------------------------------------------------------------------

// sum of floor((a i + b) / m) for i < n (a, b >= 0): the points under a line,
// counted by the Euclidean algorithm.
__device__ __forceinline__ long long floor_sum(long long n, long long m, long long a, long long b) {
    long long s = 0;
    while (n > 0) {
        s += (a / m) * (n * (n - 1) / 2) + (b / m) * n;
        a %= m;
        b %= m;
        const long long top = a * n + b;
        if (top < m) break;
        n = top / m;
        b = top % m;
        const long long t = m;
        m = a;
        a = t;
    }
    return s;
}

// A sequence's row blocks: block rb has tiles(rb) position tiles,
// floor((step rb + base) / div) but for the last block.
struct Blocks {
    int nrb, last;
    long long step, base, div;
    __device__ __forceinline__ int tiles(int rb) const {
        return rb == nrb - 1 ? last : (int)((step * rb + base) / div);
    }
    __device__ __forceinline__ long long before(int rb) const { return floor_sum(min(rb, nrb - 1), div, step, base) + (rb == nrb ? last : 0); }
};
__device__ __forceinline__ Blocks blocks_of(const Seq &s, int group) {
    Blocks b;
    b.nrb = (int)(((long long)s.nq * group + kBlockRows - 1) / kBlockRows);
    b.last = max(1, (s.len + kPos - 1) / kPos);
    if (s.nq > s.len) { // some rows see nothing: every block as long as the last
        b.step = 0, b.base = b.last, b.div = 1;
    } else { // its last row's position, + 1: len - nq + 1 + floor((256 rb + 255) / group)
        b.step = kBlockRows;
        b.base = (long long)(s.len - s.nq + 1) * group + kBlockRows - 1 + (long long)(kPos - 1) * group;
        b.div = (long long)kPos * group;
    }
    return b;
}

struct Where { // a segment and a position tile of it
    int i, head, rb, tile, tiles;
    Seq s;
    Blocks b;
    long long from; // the segment's first position tile in the list
};

__device__ __forceinline__ Seq prompt_seq(const Params &p, int i) {
    Seq s = seq_at(p, p.a.starts, p.a.lens, i);
    if (s.nq <= p.rows_cut / p.group) s.nq = 0; // the other kernel's
    return s;
}

// sums[e] = position tiles of the sequences before entry e, for all threads of a block; the total.
template <int NT> __device__ __forceinline__ long long list_sums(const Params &p, long long *sums) {
    constexpr int NW = NT / 32, PER = (kKvSums + NT - 1) / NT;
    __shared__ long long scan[NW];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n = p.a.n, entries = (n + (1 << p.shift_sums) - 1) >> p.shift_sums;
    long long own[PER], sum = 0;
#pragma unroll
    for (int u = 0; u < PER; u++) {
        const int e = tid * PER + u;
        own[u] = 0;
        if (e < entries)
            for (int i = e << p.shift_sums; i < min(n, (e + 1) << p.shift_sums); i++) {
                const Seq s = prompt_seq(p, i);
                if (s.nq == 0) continue;
                const Blocks b = blocks_of(s, p.group);
                own[u] += b.before(b.nrb) * p.c.n_kv;
            }
        sum += own[u];
    }
    long long inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
    }
    if (lane == 31) scan[warp] = inc;
    __syncthreads();
    long long before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < NW; w++) {
        if (w < warp) before += scan[w];
        total += scan[w];
    }
    before += inc - sum;
#pragma unroll
    for (int u = 0; u < PER; u++) {
        const int e = tid * PER + u;
        if (e < entries) sums[e] = before;
        before += own[u];
    }
    if (tid == 0) sums[entries] = total;
    __syncthreads();
    return total;
}

// The segment that holds position tile x of the list; called by whole warps.
__device__ __forceinline__ Where find(const Params &p, const long long *sums, long long x) {
    const int lane = threadIdx.x & 31;
    const int entries = (p.a.n + (1 << p.shift_sums) - 1) >> p.shift_sums;
    Where w;
    int lo = 0, hi = entries;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (sums[mid] <= x)
            lo = mid;
        else
            hi = mid;
    }
    long long rest = x - sums[lo], per = 0;
    for (w.i = lo << p.shift_sums; w.i < p.a.n; w.i++) {
        w.s = prompt_seq(p, w.i);
        if (w.s.nq == 0) continue;
        w.b = blocks_of(w.s, p.group);
        per = w.b.before(w.b.nrb);
        if (rest < per * p.c.n_kv) break;
        rest -= per * p.c.n_kv;
    }
    w.head = (int)(rest / per);
    rest -= per * w.head;
    // the last row block that starts at or before `rest`: 32 candidates at a time
    int a = 0, z = w.b.nrb; // before(a) <= rest < before(z)
    while (z - a > 1) {
        const int stride = (z - a + 31) / 32, c = min(z, a + lane * stride);
        const unsigned ok = __ballot_sync(0xffffffffu, w.b.before(c) <= rest);
        const int k = 31 - __clz(ok);
        const int na = min(z, a + k * stride);
        z = min(z, na + stride);
        a = na;
    }
    w.rb = a;
    w.tile = (int)(rest - w.b.before(a));
    w.tiles = w.b.tiles(a);
    w.from = x - w.tile;
    return w;
}

__device__ __forceinline__ void next_segment(const Params &p, Where &w) {
    w.from += w.tiles;
    w.tile = 0;
    if (++w.rb == w.b.nrb) {
        w.rb = 0;
        if (++w.head == p.c.n_kv) {
            w.head = 0;
            while (++w.i < p.a.n) {
                w.s = prompt_seq(p, w.i);
                if (w.s.nq) break;
            }
            if (w.i >= p.a.n) return;
            w.b = blocks_of(w.s, p.group);
        }
    }
    w.tiles = w.b.tiles(w.rb);
}

// Positions that row `row` of the sequence sees.
__device__ __forceinline__ int sees(const Seq &s, int row, int group) {
    return min(s.len, max(0, s.len - s.nq + row / group + 1));
}
// Position tiles of the segment's row tile t (0: A, 1: B): 0 without rows.
__device__ __forceinline__ int tiles_of(const Where &w, int t, int group) {
    const int first = w.rb * kBlockRows + t * kRows, rows = w.s.nq * group;
    if (first >= rows) return 0;
    return max(1, (sees(w.s, min(rows, first + kRows) - 1, group) + kPos - 1) / kPos);
}

// ---- tensor memory and MMA -------------------------------------------------------------

__device__ __forceinline__ void tmem_ld32(uint32_t a, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(a)
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t a, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(a),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
        "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
        "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t a, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
                     a),
                 "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
                 "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D (f32, TMEM) += A B, A and B float16 and K-major; N columns.
__device__ __forceinline__ constexpr uint32_t idesc_f16(int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
}
// The operand descriptor at a shared-memory address: 128-byte rows, swizzled, 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t desc(uint32_t addr) { return tqp::umma_desc(addr, 16, 1024, 2); }
// Byte of 16-byte chunk c of row r in such an operand.
__device__ __forceinline__ uint32_t chunk_at(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

struct Shared { // static shared memory
    uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
    uint64_t q_ready[2], s_full[2], p_ready[2], o_full[2];
    float f[kConsts][kBlocks], lv[kConsts][kBlocks], rv[kConsts][kBlocks];
    uint32_t tmem;
    volatile int late;
};

template <int HDP, int PIECES, typename T>
__global__ void __launch_bounds__(kThreads, 1) kv_prompt_kernel(const __grid_constant__ Params p) {
    constexpr int ST = stages_of(HDP, PIECES);
    constexpr uint32_t OP = (uint32_t)operand_bytes(HDP);
    extern __shared__ unsigned char raw[];
    __shared__ __align__(16) Shared sh;
    unsigned char *base = reinterpret_cast<unsigned char *>(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    unsigned char *Qs = base;                       // [2 tiles][PIECES][OP]
    unsigned char *Ks = Qs + 2 * PIECES * OP;       // [ST][OP]
    unsigned char *Vs = Ks + ST * OP;               // [ST][OP]
    long long *sums = reinterpret_cast<long long *>(Vs + ST * OP);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int group = p.group;
    const long long total = list_sums<kThreads>(p, sums);
    const int G = (int)min((long long)gridDim.x, (total + kMinTiles - 1) / kMinTiles);
    if ((int)blockIdx.x >= G) return; // none: G = 0
    const TqSplit split(total, G);
    const long long x0 = split.start(blockIdx.x), x1 = split.start(blockIdx.x + 1);

    if (tid == 0) {
        for (int s = 0; s < 2; s++) {
            tqp::mbar_init(&sh.k_full[s], kConvThreads);
            tqp::mbar_init(&sh.v_full[s], kConvThreads);
            tqp::mbar_init(&sh.k_empty[s], 1);
            tqp::mbar_init(&sh.v_empty[s], 1);
            tqp::mbar_init(&sh.q_ready[s], kRows);
            tqp::mbar_init(&sh.p_ready[s], kRows);
            tqp::mbar_init(&sh.s_full[s], 1);
            tqp::mbar_init(&sh.o_full[s], 1);
        }
        sh.late = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                         tqp::smem_u32(&sh.tmem))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tqp::tc_fence_before();
    __syncthreads();
    tqp::tc_fence_after();
    const uint32_t tmem = sh.tmem;
    // columns: S of A, S of B (P over them), O of A, O of B
    auto s_col = [&](int t) { return tmem + t * kPos; };
    auto o_col = [&](int t) { return tmem + 2 * kPos + t * HDP; };

    Where w = find(p, sums, x0);
    long long x = x0; // position tiles of the list done

    if (warp < kSoftWarps) {
        // ================= softmax: thread = row of tile t =================
        const int t = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_at = s_col(t) + lanes, o_at = o_col(t) + lanes;
        unsigned tick = 0, s_phase = 0, o_phase = 0; // position tiles of the CTA so far; barrier phases
        while (x < x1) {
            const int cnt = (int)min((long long)(w.tiles - w.tile), x1 - x);
            const int mine = min(cnt, max(0, tiles_of(w, t, group) - w.tile));
            const int rows = w.s.nq * group, r = w.rb * kBlockRows + t * kRows + row;
            const int tok = r / group, hq = w.head * group + r - tok * group;
            const bool live = r < rows;
            const int lim = live ? sees(w.s, r, group) : w.s.len;
            float M = -INFINITY, L = 0.f;
            if (mine > 0) {
                // ---- this row of Q, as float16 pieces ----
                const T *q = static_cast<const T *>(p.a.q) + (size_t)(w.s.start + tok) * p.a.q_stride + (size_t)hq * p.c.hd;
                float big = 0.f;
                for (int d = 0; d < HDP; d += 8) {
                    float y[8];
                    if (live && d < p.c.hd) {
                        load8(q + d, p.vec, y);
#pragma unroll
                        for (int u = 0; u < 8; u++) big = fmaxf(big, fabsf(y[u]));
                    }
                }
                float back;
                float unit = row_scale(big, &back);
                if (p.scale2 < 0.f) unit = -unit; // the block factors stay positive
                unsigned char *qs = Qs + t * PIECES * OP;
                for (int c = 0; c < HDP / 8; c++) {
                    float y[8];
                    if (live && 8 * c < p.c.hd)
                        load8(q + 8 * c, p.vec, y);
                    else
#pragma unroll
                        for (int u = 0; u < 8; u++) y[u] = 0.f;
                    unsigned hi[4], lo[4];
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        const float a = y[2 * u] * unit, b = y[2 * u + 1] * unit;
                        hi[u] = pack2(a, b);
                        const float2 h = unpack2(hi[u]);
                        lo[u] = pack2(a - h.x, b - h.y);
                    }
                    const uint32_t at = (c >> 3) * (kRows * 128) + chunk_at(row, c & 7);
                    *reinterpret_cast<uint4 *>(qs + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    if (PIECES == 2) *reinterpret_cast<uint4 *>(qs + OP + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
                tqp::fence_proxy_async();
                tqp::tc_fence_before(); // the last segment's reads of S and O
                tqp::mbar_arrive(&sh.q_ready[t]);

                for (int j = 0; j < mine; j++) {
                    const int pos0 = (w.tile + j) * kPos, cs = (tick + j) % kConsts;
                    wait_slot(&sh.s_full[t], s_phase & 1, &sh.late, p.c.status);
                    s_phase++;
                    tqp::tc_fence_after();
                    const int seen = lim - pos0; // columns below it are visible
                    const bool whole = __all_sync(0xffffffffu, seen >= kPos);
                    // ---- M ----
                    float top = -INFINITY;
#pragma unroll 1
                    for (int c = 0; c < 4; c++) {
                        uint32_t v[32];
                        tmem_ld32(s_at + 32 * c, v);
                        tqp::tmem_wait_ld();
#pragma unroll
                        for (int b = 0; b < 2; b++) {
                            float mx = -INFINITY;
#pragma unroll
                            for (int u = 0; u < 16; u++) {
                                float s = __uint_as_float(v[16 * b + u]);
                                if (!whole) s = 32 * c + 16 * b + u < seen ? s : -INFINITY;
                                mx = fmaxf(mx, s);
                            }
                            top = fmaxf(top, fmaf(mx, sh.f[cs][2 * c + b] * back, sh.lv[cs][2 * c + b]));
                        }
                    }
                    float alpha = 1.f;
                    if (top > M + kSlack || (M == -INFINITY && top > M)) {
                        alpha = ex2(M - top);
                        M = top;
                        L *= alpha;
                    }
                    if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
                        // S of this tile is complete, so O += P V of the last one is (issued before it)
#pragma unroll 1
                        for (int c = 0; c < HDP / 32; c++) {
                            uint32_t v[32];
                            tmem_ld32(o_at + 32 * c, v);
                            tqp::tmem_wait_ld();
#pragma unroll
                            for (int u = 0; u < 32; u++) v[u] = __float_as_uint(__uint_as_float(v[u]) * alpha);
                            tmem_st32(o_at + 32 * c, v);
                        }
                    }
                    const float use = M == -INFINITY ? 0.f : M - kUnit;
                    // ---- P over S ----
#pragma unroll 1
                    for (int c = 0; c < 4; c++) {
                        uint32_t v[32], hi[16], lo[16];
                        tmem_ld32(s_at + 32 * c, v);
                        tqp::tmem_wait_ld();
#pragma unroll
                        for (int b = 0; b < 2; b++) {
                            const float fb = sh.f[cs][2 * c + b] * back, ob = sh.lv[cs][2 * c + b] - use;
                            float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                            for (int u = 0; u < 16; u += 2) {
                                const float2 s = make_float2(__uint_as_float(v[16 * b + u]), __uint_as_float(v[16 * b + u + 1]));
                                const float2 e = __ffma2_rn(s, make_float2(fb, fb), make_float2(ob, ob));
                                float2 y = make_float2(ex2(e.x), ex2(e.y));
                                if (!whole) { // 0 whatever the block's scales are
                                    y.x = 32 * c + 16 * b + u < seen ? y.x : 0.f;
                                    y.y = 32 * c + 16 * b + u + 1 < seen ? y.y : 0.f;
                                }
                                sum = __fadd2_rn(sum, y);
                                const unsigned h = pack2(y.x, y.y);
                                hi[8 * b + u / 2] = h;
                                if (PIECES == 2) {
                                    const float2 z = unpack2(h);
                                    lo[8 * b + u / 2] = pack2(y.x - z.x, y.y - z.y);
                                }
                            }
                            L = fmaf(sum.x + sum.y, sh.rv[cs][2 * c + b], L);
                        }
                        if (PIECES == 1) {
                            tmem_st16(s_at + 16 * c, hi);
                        } else {
                            tmem_st16(s_at + 32 * c, hi);
                            tmem_st16(s_at + 32 * c + 16, lo);
                        }
                    }
                    tmem_wait_st();
                    tqp::tc_fence_before();
                    tqp::mbar_arrive(&sh.p_ready[t]);
                }
                wait_slot(&sh.o_full[t], o_phase & 1, &sh.late, p.c.status);
                o_phase++;
                tqp::tc_fence_after();
            }
            // ---- out, or this part of it ----
            const bool all = w.from >= x0 && w.from + w.tiles <= x1;
            if (all) {
                const float inv = L == 0.f ? 0.f : 1.f / L;
                T *o = static_cast<T *>(p.a.out) + (size_t)(w.s.start + tok) * p.a.out_stride + (size_t)hq * p.c.hd;
                if (mine > 0)
#pragma unroll 1
                    for (int c = 0; c < HDP / 32; c++) {
                        uint32_t v[32];
                        tmem_ld32(o_at + 32 * c, v);
                        tqp::tmem_wait_ld();
                        if (live)
#pragma unroll
                            for (int u = 0; u < 32; u += 8)
                                if (32 * c + u < p.c.hd) {
                                    float y[8];
#pragma unroll
                                    for (int e = 0; e < 8; e++) y[e] = __uint_as_float(v[u + e]) * inv;
                                    store8(o + 32 * c + u, p.vec, y);
                                }
                    }
            } else {
                float *part = reinterpret_cast<float *>(static_cast<char *>(p.a.workspace) + kKvHead) +
                              ((size_t)blockIdx.x * 2 + (w.from >= x0 ? 1 : 0)) * partial_floats(HDP);
                const int pr = t * kRows + row;
                if (mine > 0)
#pragma unroll 1
                    for (int c = 0; c < HDP / 32; c++) {
                        uint32_t v[32];
                        tmem_ld32(o_at + 32 * c, v);
                        tqp::tmem_wait_ld();
#pragma unroll
                        for (int u = 0; u < 32; u += 4)
                            *reinterpret_cast<uint4 *>(part + (size_t)pr * HDP + 32 * c + u) =
                                make_uint4(v[u], v[u + 1], v[u + 2], v[u + 3]);
                    }
                part[kBlockRows * HDP + pr] = mine > 0 ? M : __int_as_float(0x7f800001); // a NaN: no part here
                part[kBlockRows * HDP + kBlockRows + pr] = L;
            }
            x += cnt;
            tick += cnt;
            if (x < x1) next_segment(p, w);
        }
    } else if (warp < kMmaWarp) {
        // ================= codes -> float16 operands =================
        const int ct = tid - 32 * kSoftWarps;
        constexpr int U = kPos * HDP / 16 / kConvThreads; // 16-byte words per thread and tile
        constexpr int PER_ROW = HDP / 16;
        // the segment and tile that is loaded (ahead of what is converted)
        Where ld = w;
        long long lx = x0;
        int lt = w.tile;
        int id = -1; // lanes 0..7: the page of block `lane` of the tile being loaded
        float2 sc = make_float2(0.f, 0.f), sc_keys;
        uint4 rk[U], rv[U];
        const float mag = fabsf(p.scale2);
        auto fetch = [&]() {
            id = -1;
            sc = make_float2(-1.f, 0.f);
            if (lx >= x1 || lane >= kBlocks) return;
            const int pos = lt * kPos + lane * TQ_KV_BLOCK;
            const int rows = ld.s.nq * group;
            if (pos < sees(ld.s, min(rows, (ld.rb + 1) * kBlockRows) - 1, group)) {
                id = p.a.table[(size_t)ld.i * p.a.table_stride + (pos >> p.c.page_shift)];
                if (id < 0 || id >= p.c.n_pages) {
                    id = -1;
                    atomicOr(p.c.status, TQ_KV_STATUS_PAGE);
                } else {
                    sc = __ldg(p.c.scale + (size_t)id * p.c.n_kv + ld.head);
                }
            }
        };
        // word u of the thread: of block blk(u); keys: its row and chunk, values: its dimension
        auto load = [&](const int8_t *from, uint4 (&r)[U], bool values) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int word = ct + u * kConvThreads, blk = word / HDP, in = word - blk * HDP; // HDP words a block
                const int page = __shfl_sync(0xffffffffu, id, blk);
                const float c = __shfl_sync(0xffffffffu, sc.y, blk);
                r[u] = make_uint4(0, 0, 0, 0);
                if (page >= 0 && !(values && c == 0.f)) {
                    const int b = ((lt * kPos + blk * TQ_KV_BLOCK) & (p.c.page - 1)) >> 4;
                    r[u] = __ldg(reinterpret_cast<const uint4 *>(from + kv_block_offset(p.c, page, ld.head, b)) + in);
                }
            }
        };
        auto expand = [&](const uint4 &r, uint4 &lo, uint4 &hi) {
            cvt4(r.x, lo.x, lo.y);
            cvt4(r.y, lo.z, lo.w);
            cvt4(r.z, hi.x, hi.y);
            cvt4(r.w, hi.z, hi.w);
        };
        auto step = [&]() { // to the next tile to be loaded
            lx++;
            lt++;
            if (lx < x1 && lt == ld.tiles) {
                next_segment(p, ld);
                lt = 0;
            }
        };
        static_assert(kPos * HDP / 16 == HDP * kBlocks, "a block is HDP words of 16 bytes");
        fetch();
        load(p.c.k, rk, false);
        unsigned k = 0;
        const unsigned count = (unsigned)(x1 - x0);
        for (k = 0; k < count; k++) {
            const unsigned s = k % ST, round = k / ST;
            sc_keys = sc;
            load(p.c.v, rv, true);
            // ---- keys of tile k ----
            if (round > 0) wait_slot(&sh.k_empty[s], (round - 1) & 1, &sh.late, p.c.status);
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int word = ct + u * kConvThreads, r = word / PER_ROW, c = word - r * PER_ROW;
                // where the cache keeps chunk c of the row (tq_kv.h): here the word is chunk c as stored
                const int chunk = HDP >= 128 ? c ^ ((r & 1) << 2) : c; // 16 dimensions
                uint4 a, b;
                expand(rk[u], a, b);
                unsigned char *to = Ks + s * OP + (chunk >> 2) * (kPos * 128);
                const int c0 = 2 * (chunk & 3), h = HDP >= 128 ? chunk >> 2 & 1 : 0; // two halves in turn: distinct banks
                *reinterpret_cast<uint4 *>(to + chunk_at(r, c0 + h)) = h ? b : a;
                *reinterpret_cast<uint4 *>(to + chunk_at(r, c0 + 1 - h)) = h ? a : b;
            }
            if (ct < kBlocks) { // the scales of the tile's blocks; x < 0: a block that is not there
                const bool there = sc_keys.x >= 0.f || sc_keys.x != sc_keys.x;
                const bool plain = sc_keys.y > 0.f;
                sh.f[k % kConsts][ct] = there ? sc_keys.x * mag : 0.f;
                sh.lv[k % kConsts][ct] = !there ? -INFINITY : plain ? log2f(sc_keys.y) : sc_keys.y == 0.f ? 0.f : sc_keys.y;
                sh.rv[k % kConsts][ct] = !there ? 0.f : plain ? 1.f / sc_keys.y : 1.f;
            }
            tqp::fence_proxy_async();
            tqp::mbar_arrive(&sh.k_full[s]);
            step();
            fetch();
            load(p.c.k, rk, false);
            // ---- values of tile k ----
            if (round > 0) wait_slot(&sh.v_empty[s], (round - 1) & 1, &sh.late, p.c.status);
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int word = ct + u * kConvThreads, blk = word / HDP, d = word - blk * HDP;
                uint4 a, b;
                expand(rv[u], a, b);
                unsigned char *to = Vs + s * OP + (blk >> 2) * (HDP * 128);
                *reinterpret_cast<uint4 *>(to + chunk_at(d, 2 * (blk & 3))) = a;
                *reinterpret_cast<uint4 *>(to + chunk_at(d, 2 * (blk & 3) + 1)) = b;
            }
            tqp::fence_proxy_async();
            tqp::mbar_arrive(&sh.v_full[s]);
        }
    } else {
        // ================= MMA issue: one thread =================
        if (lane == 0) {
            unsigned tick = 0, q_phase[2] = {0, 0}, p_phase[2] = {0, 0};
            const uint32_t q0 = tqp::smem_u32(Qs), k0 = tqp::smem_u32(Ks), v0 = tqp::smem_u32(Vs);
            auto scores = [&](int t, unsigned n) { // S(t) = Q(t) K(n)^T
                const uint32_t kb = k0 + (n % ST) * OP;
#pragma unroll
                for (int pc = 0; pc < PIECES; pc++)
#pragma unroll
                    for (int ks = 0; ks < HDP / 16; ks++) {
                        const uint32_t o = (ks >> 2) * (kRows * 128) + (ks & 3) * 32;
                        mma_ss(s_col(t), desc(q0 + (t * PIECES + pc) * OP + o), desc(kb + o), idesc_f16(kPos),
                               pc > 0 || ks > 0);
                    }
                tqp::umma_commit(&sh.s_full[t]);
            };
            auto products = [&](int t, unsigned n, bool first) { // O(t) += P(t) V(n)
                const uint32_t vb = v0 + (n % ST) * OP;
#pragma unroll
                for (int pc = 0; pc < PIECES; pc++)
#pragma unroll
                    for (int ks = 0; ks < kPos / 16; ks++) {
                        const uint32_t a = PIECES == 1 ? s_col(t) + 8 * ks : s_col(t) + 32 * (ks >> 1) + 16 * pc + 8 * (ks & 1);
                        mma_ts(o_col(t), a, desc(vb + (ks >> 2) * (HDP * 128) + (ks & 3) * 32), idesc_f16(HDP),
                               !first || pc > 0 || ks > 0);
                    }
            };
            while (x < x1) {
                const int cnt = (int)min((long long)(w.tiles - w.tile), x1 - x);
                int mine[2];
#pragma unroll
                for (int t = 0; t < 2; t++) mine[t] = min(cnt, max(0, tiles_of(w, t, group) - w.tile));
                for (int j = -1; j < cnt; j++) {
                    const unsigned n = tick + j;
                    for (int t = 0; t < 2; t++) {
                        // every tile's operands are waited for once, whether a row tile uses them or not
                        if (j >= 0 && t == 0) wait_slot(&sh.v_full[n % ST], (n / ST) & 1, &sh.late, p.c.status);
                        if (j >= 0 && j < mine[t]) {
                            wait_slot(&sh.p_ready[t], p_phase[t]++ & 1, &sh.late, p.c.status);
                            tqp::tc_fence_after();
                            products(t, n, j == 0);
                            if (j + 1 == mine[t]) tqp::umma_commit(&sh.o_full[t]);
                        }
                        if (j >= 0 && t == 1) tqp::umma_commit(&sh.v_empty[n % ST]);
                        if (j + 1 < cnt && t == 0)
                            wait_slot(&sh.k_full[(n + 1) % ST], ((n + 1) / ST) & 1, &sh.late, p.c.status);
                        if (j + 1 < mine[t]) {
                            if (j < 0) wait_slot(&sh.q_ready[t], q_phase[t]++ & 1, &sh.late, p.c.status);
                            tqp::tc_fence_after();
                            scores(t, n + 1);
                        }
                        if (j + 1 < cnt && t == 1) tqp::umma_commit(&sh.k_empty[(n + 1) % ST]);
                    }
                }
                x += cnt;
                tick += cnt;
                if (x < x1) next_segment(p, w);
            }
        }
    }
    __syncwarp();
    tqp::tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tqp::tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// Joins the parts of the segment that CTA blockIdx.x of the kernel above began
// and did not end: 32 rows a block.
template <int HDP, typename T>
__global__ void __launch_bounds__(kJoinThreads) kv_join_kernel(const __grid_constant__ Params p, int grid) {
    __shared__ long long sums[kKvSums + 1];
    const long long total = list_sums<kJoinThreads>(p, sums);
    const int G = (int)min((long long)grid, (total + kMinTiles - 1) / kMinTiles);
    const int cta = blockIdx.x;
    if (cta + 1 >= G) return;
    const TqSplit split(total, G);
    const long long c0 = split.start(cta), c1 = split.start(cta + 1);
    const Where w = find(p, sums, c1 - 1);
    if (w.from < c0 || w.from + w.tiles <= c1) return; // another CTA's, or whole
    const int k = split.owner(w.from + w.tiles - 1) - cta + 1;
    const float *part = reinterpret_cast<const float *>(static_cast<const char *>(p.a.workspace) + kKvHead);
    auto at = [&](int j) { return part + ((size_t)(cta + j) * 2 + (j == 0 ? 1 : 0)) * partial_floats(HDP); };
    const int rows = min(kBlockRows, w.s.nq * p.group - w.rb * kBlockRows);
    constexpr int Q4 = HDP / 4;
    for (int e = threadIdx.x; e < kJoinRows * Q4; e += kJoinThreads) {
        const int r = blockIdx.y * kJoinRows + e / Q4, d = (e % Q4) * 4;
        if (r >= rows || d >= p.c.hd) continue;
        float M = -INFINITY;
        for (int j = 0; j < k; j++) M = fmaxf(M, __ldcg(at(j) + kBlockRows * HDP + r)); // NaN: no part, passed over
        const float use = M == -INFINITY ? 0.f : M;
        float L = 0.f;
        float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int j = 0; j < k; j++) {
            const float *f = at(j);
            const float m = __ldcg(f + kBlockRows * HDP + r);
            if (m != m) continue;
            const float g = exp2f(m - use);
            const float4 y = __ldcg(reinterpret_cast<const float4 *>(f + (size_t)r * HDP + d));
            L = fmaf(g, __ldcg(f + kBlockRows * HDP + kBlockRows + r), L);
            A.x = fmaf(g, y.x, A.x);
            A.y = fmaf(g, y.y, A.y);
            A.z = fmaf(g, y.z, A.z);
            A.w = fmaf(g, y.w, A.w);
        }
        const float inv = L == 0.f ? 0.f : 1.f / L;
        const int row = w.rb * kBlockRows + r, tok = row / p.group, hq = w.head * p.group + row - tok * p.group;
        T *o = static_cast<T *>(p.a.out) + (size_t)(w.s.start + tok) * p.a.out_stride + (size_t)hq * p.c.hd + d;
        Elem<T>::put2(o, A.x * inv, A.y * inv, p.vec, true);
        Elem<T>::put2(o + 2, A.z * inv, A.w * inv, p.vec, true);
    }
}

template <int HDP, int PIECES, typename T> cudaError_t launch(const Params &p, int sms, cudaStream_t st) {
    static TqDeviceOnce once;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess)
        e = tq_device_once(once, dev, [] {
            return cudaFuncSetAttribute(kv_prompt_kernel<HDP, PIECES, T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        (int)smem_bytes(HDP, PIECES));
        });
    if (e != cudaSuccess) return e;
    kv_prompt_kernel<HDP, PIECES, T><<<sms, kThreads, smem_bytes(HDP, PIECES), st>>>(p);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    kv_join_kernel<HDP, T><<<dim3(sms, kBlockRows / kJoinRows), kJoinThreads, 0, st>>>(p, sms);
    return cudaGetLastError();
}

} // namespace

size_t tq_kv_prompt_workspace(int hdp, int sms) {
    return hdp > 128 ? 0 : kKvHead + (size_t)sms * 2 * partial_floats(hdp) * sizeof(float);
}

cudaError_t tq_kv_launch_prompt(const TqKvParams &p, int sms, cudaStream_t st) {
    if (p.c.hdp == 64) {
        if (p.a.dtype == TQ_LINEAR_F32) return launch<64, 2, float>(p, sms, st);
        if (p.a.dtype == TQ_LINEAR_F16) return launch<64, 1, __half>(p, sms, st);
        return launch<64, 1, __nv_bfloat16>(p, sms, st);
    }
    if (p.a.dtype == TQ_LINEAR_F32) return launch<128, 2, float>(p, sms, st);
    if (p.a.dtype == TQ_LINEAR_F16) return launch<128, 1, __half>(p, sms, st);
    return launch<128, 1, __nv_bfloat16>(p, sms, st);
}
