// tq_kv_prompt.cu — attention of many query rows over the paged 8-bit cache on
// the 5th-generation tensor cores (the formulas are in tq_kv_attn.cu; head sizes
// up to 128; sequences of more than tokens_cut new tokens).
//
// The rows of a sequence and KV head (new tokens x query heads of the group) are
// cut into blocks of 256, two tiles A and B of 128 rows, positions into tiles of
// 128. For each position tile and row tile:
//   S = Q K^T    tcgen05.mma kind::f16, operands in shared memory, S in TMEM;
//   softmax      two threads a row: S from TMEM, P back over S as float16;
//   O += P V     tcgen05.mma with P from TMEM, O in TMEM.
// While the softmax of one row tile runs, the tensor cores work for the other.
// Codes become float16 once per CTA and position tile (exact), in four warps
// that go through registers: HBM/L2 -> codes -> float16 -> swizzled operand.
// Float32 queries take two float16 pieces of q and of p (22 bits): twice the
// products. 16-bit queries take one, which holds q exactly and rounds p to 11 bits:
// off by at most 2^-11, an eighth of a bfloat16 output's own rounding and as much
// as a float16 output's, but averaged over the positions. Against 64 bits the error
// (2-norm) is 1.7e-3 with one piece or two in bfloat16, 2.3e-4 and 2.1e-4 in
// float16; two pieces of p cost whole prompts 241 us in place of 211, mixed
// batches 184 in place of 165 (whole calls).
//
// The scales. With a_b, c_b the key and value scale of a 16-position block,
//   w_t = s_t a_b + log2 c_b,  M = max w_t - 10 (raised only when w exceeds M + 14),
//   P = 2^(w_t - M),  O = sum P v codes,  L = sum_b (sum P) / c_b,
//   out = O / L:
// the value scale rides in the exponent at no cost, and P stays below 2^14. A
// block of value scale below 2^-92 counts with c = 2^-60 and zero codes: low enough
// for the bits of what has values, high enough for its own share of L.
//
// Work: (sequence, KV head, row block) segments laid end to end, each as long as
// its position tiles and kSegCost units before them (its queries come in and its
// outputs go out), and cut evenly over one CTA per SM. A cut segment's parts go to
// the workspace; the second kernel joins them in order (the same bits each time).
// Cost 2: 122 GFLOP of whole prompts took 204 us, mixed sequences of 73 GFLOP 161;
// cost 1: 226 and 168; 3: 205 and 161; none: 265 and 265. (All before w was rounded
// apart from its difference to M, as the sides below: 212 and 163 since.)
//
// Roles. Two softmax threads a row (211 us; one 217), sixteen warps; four that
// widen codes (they are busy 60% of the time); one that issues; one that finds
// segments, pages and scales up to three tiles ahead. Barriers are arrived at once
// a warp (204 us; by every thread 208).
//
// Bound by the chain of one row tile, scores - maximum - exponentials - product,
// whose parts other tiles only partly cover: whole prompts in bfloat16 run at 575
// TFLOP/s (35% of the measured matmul rate), the tensor pipe 32%, the exponential
// unit 34%, issue slots 55% used. Tried: P before the row's maximum is known, in one
// pass over S (264 us, its code is too long for the instruction caches), the issuing
// warp kept together (206), S read 32 columns at a time (204, the same).
#include <climits>
#include <type_traits>

#include "tq_kv_attn.cuh"

namespace {

using namespace tqkv;
using Params = TqKvParams;

constexpr int kRows = 128;      // rows of a tile
constexpr int kBlockRows = 256; // rows of a block: tiles A and B
constexpr int kPos = 128;       // positions of a tile
constexpr int kBlocks = kPos / TQ_KV_BLOCK;
constexpr int kSoftWarps = 16, kConvWarps = 4;
constexpr int kTileThreads = 2 * kRows; // softmax threads of a row tile: two a row, half the columns each
constexpr int kConvThreads = 32 * kConvWarps;
constexpr int kMmaWarp = kSoftWarps + kConvWarps; // one thread of it issues; the next warp loads
constexpr int kThreads = 32 * (kMmaWarp + 2);
constexpr int kConsts = 4;      // position tiles whose scales are kept
constexpr int kSegCost = 2;     // what a segment costs besides its position tiles, in position tiles
constexpr int kMinUnits = 3;    // units per CTA below which fewer CTAs work
constexpr float kUnit = 10.f;   // log2 of P where w is the row's largest
constexpr float kMostP = 14.f;  // and what it may grow to before M is raised
constexpr int kJoinThreads = 256, kJoinRows = 32;

constexpr size_t kSharedRoom = 3 * 1024; // struct Shared, behind the operands
constexpr int stages_of(int hdp, int pieces) { return hdp == 128 && pieces == 2 ? 1 : 2; }
constexpr size_t operand_bytes(int hdp) { return (size_t)kPos * hdp * 2; } // a K or V tile, or a piece of a Q tile
constexpr size_t smem_bytes(int hdp, int pieces) {
    return kSharedRoom + operand_bytes(hdp) * (2 * pieces + 2 * stages_of(hdp, pieces) + 1); // the staged codes are one more
}
constexpr size_t partial_floats(int hdp) { return (size_t)kBlockRows * (hdp + 2); }

// ---- the list of work ------------------------------------------------------------------

// A sequence's row blocks. Block rb's last row is of new token (256 rb + 255) /
// group, so it sees `first` + that many positions; the last block sees them all.
struct Blocks {
    int nrb, last;
    unsigned first; // 0: every block like the last (some rows see nothing)
    __device__ __forceinline__ int tiles(int rb, int group) const {
        if (rb == nrb - 1 || first == 0) return last;
        return (int)((first + (unsigned)(rb * kBlockRows + kBlockRows - 1) / (unsigned)group + kPos - 1) / kPos);
    }
};
__device__ __forceinline__ Blocks blocks_of(const Seq &s, int group) {
    Blocks b;
    b.nrb = (s.nq * group + kBlockRows - 1) / kBlockRows;
    b.last = max(1, (int)(((unsigned)s.len + kPos - 1) / kPos));
    b.first = s.nq > s.len ? 0u : (unsigned)(s.len - s.nq + 1);
    return b;
}
// The units of one head, by a whole warp.
__device__ __forceinline__ long long head_units(const Blocks &b, int group) {
    long long t = 0;
    for (int rb = threadIdx.x & 31; rb < b.nrb; rb += 32) t += b.tiles(rb, group) + kSegCost;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    return t;
}

struct Where { // a segment
    int i, head, rb, tiles;
    Seq s;
    Blocks b;
    long long from; // where its position tiles begin in the list (its own cost lies before)
    // the position tiles [a, z) of it that lie in the units [x0, x1) of the list
    __device__ __forceinline__ int first(long long x0) const { return (int)min((long long)tiles, max(0ll, x0 - from)); }
};

__device__ __forceinline__ Seq prompt_seq(const Params &p, int i) {
    Seq s = seq_at(p, p.a.starts, p.a.lens, i);
    if (s.nq <= p.tokens_cut) s.nq = 0; // the other kernel's
    return s;
}

// sums[e] = units of the sequences before entry e, for all threads of a block; the total.
// scan: a word for each warp.
template <int NT> __device__ __forceinline__ long long list_sums(const Params &p, long long *sums, long long *scan) {
    constexpr int NW = NT / 32, PER = (kKvSums + NT - 1) / NT;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n = p.a.n, entries = (n + (1 << p.shift_sums) - 1) >> p.shift_sums;
    for (int e = tid; e < entries; e += NT) sums[e] = 0;
    __syncthreads();
    // 32 sequences a turn, a lane each; those of several blocks by the whole warp
    for (int i0 = warp * 32; i0 < n; i0 += NT) {
        const int i = i0 + lane;
        Seq s{0, 0, 0};
        if (i < n) s = prompt_seq(p, i);
        const Blocks b = blocks_of(s, p.group);
        long long t = s.nq && b.nrb == 1 ? b.tiles(0, p.group) + kSegCost : 0;
        for (unsigned many = __ballot_sync(0xffffffffu, s.nq && b.nrb > 1); many; many &= many - 1) {
            const int l = __ffs(many) - 1;
            const Blocks o = {__shfl_sync(0xffffffffu, b.nrb, l), __shfl_sync(0xffffffffu, b.last, l),
                              __shfl_sync(0xffffffffu, b.first, l)};
            const long long all = head_units(o, p.group);
            if (lane == l) t = all;
        }
        if (t)
            atomicAdd(reinterpret_cast<unsigned long long *>(sums + (i >> p.shift_sums)),
                      (unsigned long long)(t * p.c.n_kv));
    }
    __syncthreads();
    long long own[PER], sum = 0;
#pragma unroll
    for (int u = 0; u < PER; u++) {
        const int e = tid * PER + u;
        own[u] = e < entries ? sums[e] : 0;
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

// The segment that holds unit x of the list; called by whole warps.
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
    long long rest = x - sums[lo];
    w.head = 0;
    for (w.i = lo << p.shift_sums; w.i < p.a.n; w.i++) {
        w.s = prompt_seq(p, w.i);
        if (w.s.nq == 0) continue;
        w.b = blocks_of(w.s, p.group);
        const long long per = head_units(w.b, p.group);
        if (rest < per * p.c.n_kv) {
            for (; rest >= per; rest -= per) w.head++;
            break;
        }
        rest -= per * p.c.n_kv;
    }
    for (int r0 = 0;; r0 += 32) { // 32 row blocks at a time
        const int mine = r0 + lane < w.b.nrb ? w.b.tiles(r0 + lane, p.group) + kSegCost : 0;
        long long upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const unsigned beyond = __ballot_sync(0xffffffffu, upto > rest);
        if (beyond || r0 + 32 >= w.b.nrb) {
            const int l = beyond ? __ffs(beyond) - 1 : 31;
            w.rb = r0 + l;
            const int units = __shfl_sync(0xffffffffu, mine, l);
            w.tiles = units - kSegCost;
            w.from = x - (rest - (__shfl_sync(0xffffffffu, upto, l) - units)) + kSegCost;
            break;
        }
        rest -= __shfl_sync(0xffffffffu, upto, 31);
    }
    return w;
}

__device__ __forceinline__ void next_segment(const Params &p, Where &w) {
    w.from += w.tiles + kSegCost;
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
    w.tiles = w.b.tiles(w.rb, p.group);
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

__device__ __forceinline__ void tmem_st16(uint32_t a, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
                     a),
                 "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
                 "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t a, const uint32_t (&v)[16]) { // the first 8
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(a), "r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
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

constexpr int kSegs = 4; // segments known ahead

// A segment as the loader hands it to the other roles.
struct Seg {
    int start, nq, len; // the sequence: first token, tokens, positions
    int head, row0;     // KV head, first row
    int tile, cnt;      // position tiles tile .. tile + cnt - 1 here; cnt = 0: no more segments
    int mine[2];        // of those, how many row tiles A and B see
    int part;           // -1: the whole segment; else the workspace part
};

__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

struct Shared { // behind the operands
    uint64_t seg_full[kSegs], seg_empty[kSegs];
    uint64_t code_full[2], code_empty[2]; // staged codes: keys, values
    uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
    uint64_t q_ready[2], s_full[2], p_ready[2], o_full[2];
    Seg seg[kSegs];
    float f[kConsts][kBlocks], lv[kConsts][kBlocks], rv[kConsts][kBlocks];
    unsigned poison[kConsts]; // blocks with a scale that is not a number
    // between the two threads of a row: w, at the end L; before the first w, what its Q was divided by
    float swap[2][2][kRows];
    unsigned live[2]; // blocks of the staged keys, values that are there (values: and not all zero)
    uint32_t tmem;
    volatile int late;
};
static_assert(sizeof(Shared) <= kSharedRoom, "the room behind the operands");

template <int HDP, int PIECES, typename T>
__global__ void __launch_bounds__(kThreads, 1) kv_prompt_kernel(const __grid_constant__ Params p) {
    constexpr int ST = stages_of(HDP, PIECES);
    constexpr uint32_t OP = (uint32_t)operand_bytes(HDP), CODES = (uint32_t)kPos * HDP;
    extern __shared__ __align__(1024) unsigned char raw[];
    unsigned char *Qs = raw;                  // [2 tiles][PIECES][OP]
    unsigned char *Ks = Qs + 2 * PIECES * OP; // [ST][OP]
    unsigned char *Vs = Ks + ST * OP;         // [ST][OP]
    unsigned char *Cs = Vs + ST * OP;         // [keys, values][CODES]: as the cache holds them
    Shared &sh = *reinterpret_cast<Shared *>(Cs + 2 * CODES);
    long long *sums = reinterpret_cast<long long *>(Cs); // before the first codes
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int group = p.group;
    const long long total = list_sums<kThreads>(p, sums, sums + kKvSums + 1);
    const int G = (int)min((long long)gridDim.x, (total + kMinUnits - 1) / kMinUnits);
    if ((int)blockIdx.x >= G) return; // none: G = 0

    if (tid == 0) {
        for (int s = 0; s < kSegs; s++) {
            tqp::mbar_init(&sh.seg_full[s], 1);
            tqp::mbar_init(&sh.seg_empty[s], kSoftWarps + kConvWarps + 1);
        }
        for (int s = 0; s < 2; s++) {
            tqp::mbar_init(&sh.code_full[s], 1);
            tqp::mbar_init(&sh.code_empty[s], kConvWarps);
            tqp::mbar_init(&sh.k_full[s], kConvWarps);
            tqp::mbar_init(&sh.v_full[s], kConvWarps);
            tqp::mbar_init(&sh.k_empty[s], 1);
            tqp::mbar_init(&sh.v_empty[s], 1);
            tqp::mbar_init(&sh.q_ready[s], kTileThreads / 32);
            tqp::mbar_init(&sh.p_ready[s], kTileThreads / 32);
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
    tqp::fence_proxy_async(); // the sums: copies of codes go over them
    __syncthreads();
    tqp::tc_fence_after();
    const uint32_t tmem = sh.tmem;
    // columns: S of A, S of B (P over them), O of A, O of B
    auto s_col = [&](int t) { return tmem + t * kPos; };
    auto o_col = [&](int t) { return tmem + 2 * kPos + t * HDP; };
    auto next_seg = [&](unsigned n) -> const Seg & {
        wait_slot(&sh.seg_full[n % kSegs], (n / kSegs) & 1, &sh.late, p.c.status);
        return sh.seg[n % kSegs];
    };

    auto arrive = [&](uint64_t *bar) { // a warp's: every lane has fenced what it wrote
        __syncwarp();
        if (lane == 0) tqp::mbar_arrive(bar);
    };

    if (warp < kSoftWarps) {
        // ================= softmax: thread = half a row of tile t =================
        const int t = warp >> 3, half = warp >> 2 & 1, row = (warp & 3) * 32 + lane;
        constexpr int OC = HDP / 2; // columns of O that a thread has
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_at = s_col(t) + lanes + half * (kPos / 2), o_at = o_col(t) + lanes + half * OC;
        float *put = &sh.swap[t][half][row], *get = &sh.swap[t][1 - half][row];
        auto together = [&]() { tqp::named_sync(1 + t, kTileThreads); };
        unsigned tick = 0, s_phase = 0, o_phase = 0; // position tiles of the CTA so far; barrier phases
        for (unsigned n = 0;; n++) {
            const Seg &g = next_seg(n);
            const int cnt = g.cnt, mine = g.mine[t], tile0 = g.tile, part_at = g.part;
            if (cnt == 0) break;
            const int row0 = g.row0 + t * kRows, head = g.head, start = g.start, rows = g.nq * group;
            const int len = g.len, fresh = g.nq;
            __syncwarp();
            if (lane == 0) tqp::mbar_arrive(&sh.seg_empty[n % kSegs]);
            // a row's place among the queries or the outputs, -1 for a row that is not there
            auto place = [&](int r, long long stride) {
                const int tok = r / group, hq = head * group + r - tok * group;
                return r < rows ? (long long)(start + tok) * stride + (long long)hq * p.c.hd : -1;
            };
            const int r = row0 + row;
            const int lim = r < rows ? min(len, max(0, len - fresh + r / group + 1)) : len;
            float M = -INFINITY, L = 0.f;
            if (mine > 0) {
                // ---- Q, as float16 pieces: 16 rows a warp, each by as many lanes as it has 16-byte words.
                // The words come into the row's own memory (128 bytes for each 64 dimensions and piece)
                // and are replaced there by the pieces.
                constexpr int E = 16 / sizeof(T), LANES = HDP / E, ROWS = 32 / LANES;
                unsigned char *qs = Qs + t * PIECES * OP;
                const int word = lane % LANES, d = word * E, sub = lane / LANES, first = (warp & 7) * 16;
                const long long q_at = place(row0 + first + (lane & 15), p.a.q_stride);
                auto raw_at = [&](int qrow) {
                    return reinterpret_cast<uint4 *>(qs + (word >> 3) * (kRows * 128) + chunk_at(qrow, word & 7));
                };
                constexpr int BATCH = 4; // rows a lane works on at once
                together(); // the last segment's outputs have left this memory
                if (p.vec) {
#pragma unroll 4
                    for (int i = 0; i < 16; i += ROWS) {
                        const long long at = __shfl_sync(0xffffffffu, q_at, i + sub);
                        const bool there = at >= 0 && d < p.c.hd;
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                                         tqp::smem_u32(raw_at(first + i + sub))),
                                     "l"(static_cast<const T *>(p.a.q) + (there ? at + d : 0)), "r"(there ? 16 : 0)
                                     : "memory");
                    }
                } else {
#pragma unroll 1
                    for (int i = 0; i < 16; i += ROWS) {
                        const long long at = __shfl_sync(0xffffffffu, q_at, i + sub);
                        const bool there = at >= 0 && d < p.c.hd;
                        T *to = reinterpret_cast<T *>(raw_at(first + i + sub));
#pragma unroll 1
                        for (int e = 0; e < E; e++) to[e] = there ? static_cast<const T *>(p.a.q)[at + d + e] : T(0.f);
                    }
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                __syncwarp();
#pragma unroll 1
                for (int i = 0; i < 16; i += ROWS * BATCH) {
                    uint4 w[BATCH];
                    float big[BATCH];
#pragma unroll
                    for (int u = 0; u < BATCH; u++) w[u] = *raw_at(first + i + u * ROWS + sub);
#pragma unroll
                    for (int u = 0; u < BATCH; u++) {
                        big[u] = 0.f;
#pragma unroll
                        for (int e = 0; e < E; e++)
                            big[u] = fmaxf(big[u], fabsf(Elem<T>::get(reinterpret_cast<const T *>(&w[u]) + e)));
                    }
#pragma unroll
                    for (int o = 1; o < LANES; o <<= 1) // all lanes of a row have read their word after this
#pragma unroll
                        for (int u = 0; u < BATCH; u++) big[u] = fmaxf(big[u], __shfl_xor_sync(0xffffffffu, big[u], o));
#pragma unroll
                    for (int u = 0; u < BATCH; u++) {
                        const int qrow = first + i + u * ROWS + sub;
                        float was, unit = row_scale(big[u], &was);
                        if (p.scale2 < 0.f) unit = -unit; // the block factors stay positive
                        if (word < 2) sh.swap[t][word][qrow] = was;
                        unsigned hi[E / 2], lo[E / 2];
#pragma unroll
                        for (int e = 0; e < E / 2; e++) {
                            const float a = Elem<T>::get(reinterpret_cast<const T *>(&w[u]) + 2 * e) * unit;
                            const float b = Elem<T>::get(reinterpret_cast<const T *>(&w[u]) + 2 * e + 1) * unit;
                            hi[e] = pack2(a, b);
                            const float2 h = unpack2(hi[e]);
                            lo[e] = pack2(a - h.x, b - h.y);
                        }
                        unsigned char *to = qs + (d >> 6) * (kRows * 128) + chunk_at(qrow, (d & 63) >> 3) + 2 * (d & 7);
                        if (E == 8) {
                            *reinterpret_cast<uint4 *>(to) = make_uint4(hi[0], hi[1], hi[E / 2 - 2], hi[E / 2 - 1]);
                        } else {
                            *reinterpret_cast<uint2 *>(to) = make_uint2(hi[0], hi[1]);
                            *reinterpret_cast<uint2 *>(to + OP) = make_uint2(lo[0], lo[1]);
                        }
                    }
                }
                static_assert((sizeof(T) == 4) == (PIECES == 2), "a row's pieces take the room of its elements");
                tqp::fence_proxy_async();
                together();
                const float back = *put;
                tqp::tc_fence_before(); // the last segment's reads of S and O
                arrive(&sh.q_ready[t]);

                for (int j = 0; j < mine; j++) {
                    const int cs = (tick + j) % kConsts, b0 = half * (kBlocks / 2);
                    const int seen = lim - (tile0 + j) * kPos - half * (kPos / 2); // this half's columns below it are visible
                    const bool whole = __all_sync(0xffffffffu, seen >= kPos / 2);
                    wait_slot(&sh.s_full[t], s_phase & 1, &sh.late, p.c.status);
                    s_phase++;
                    tqp::tc_fence_after();
                    // S comes a block of 16 columns at a time, the next on its way
                    auto over = [&](auto &&use) {
                        uint32_t v0[16], v1[16];
                        tqp::tmem_ld16(s_at, v0);
                        tqp::tmem_wait_ld();
#pragma unroll 1
                        for (int b = 0; b < kBlocks / 2; b += 2) {
                            tqp::tmem_ld16(s_at + 16 * (b + 1), v1);
                            use(b, v0);
                            tqp::tmem_wait_ld();
                            if (b + 2 < kBlocks / 2) tqp::tmem_ld16(s_at + 16 * (b + 2), v0);
                            use(b + 1, v1);
                            tqp::tmem_wait_ld();
                        }
                    };
                    if (!whole) { // what a row does not see
#pragma unroll 1
                        for (int c = 0; c < kPos / 2; c += 16) {
                            uint32_t v[16];
                            tqp::tmem_ld16(s_at + c, v);
                            tqp::tmem_wait_ld();
#pragma unroll
                            for (int u = 0; u < 16; u++)
                                if (c + u >= seen) v[u] = 0xff800000u; // -inf
                            tmem_st16(s_at + c, v);
                        }
                        tmem_wait_st();
                    }
                    // a block's factor of the row's scores; never 0, for -inf times it is to stay -inf
                    auto factor = [&](int b) { return fmaxf(sh.f[cs][b0 + b] * back, kLeast); };
                    // ---- M ----
                    float top = -INFINITY;
                    over([&](int b, const uint32_t (&v)[16]) {
                        float mx = __uint_as_float(v[0]);
#pragma unroll
                        for (int u = 1; u < 15; u += 2) mx = max3(mx, __uint_as_float(v[u]), __uint_as_float(v[u + 1]));
                        mx = fmaxf(mx, __uint_as_float(v[15]));
                        top = fmaxf(top, fmaf(mx, factor(b), sh.lv[cs][b0 + b]));
                    });
                    *put = top;
                    together();
                    top = fmaxf(top, *get);
                    if (top - M > kMostP) {
                        const float next = fabsf(top) >= kFar ? top : top - kUnit; // far: M has no bits for kUnit
                        const float alpha = ex2(M - next);
                        M = next;
                        L *= alpha;
                        top = alpha;
                    } else {
                        top = 1.f;
                    }
                    if (j > 0 && __any_sync(0xffffffffu, top != 1.f)) {
                        // S of this tile is complete, so O += P V of the last one is (issued before it)
#pragma unroll 1
                        for (int c = 0; c < OC; c += 16) {
                            uint32_t o[16];
                            tqp::tmem_ld16(o_at + c, o);
                            tqp::tmem_wait_ld();
#pragma unroll
                            for (int u = 0; u < 16; u++) o[u] = __float_as_uint(__uint_as_float(o[u]) * top);
                            tmem_st16(o_at + c, o);
                        }
                    }
                    // ---- P over S: a block's 8 (or, in two pieces, 16) columns lie in columns already read ----
                    // w is rounded as the largest was, then M is taken off: from one fused product a large w could
                    // come out on either side of float16 (fused: 212 us in place of 215, and NaN or 0 from 2^24 on)
                    const float use = M == -INFINITY ? 0.f : M;
                    over([&](int b, const uint32_t (&v)[16]) {
                        uint32_t y[16];
                        const float fb = factor(b), ob = sh.lv[cs][b0 + b];
                        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                        for (int u = 0; u < 16; u += 2) {
                            const float2 s = make_float2(__uint_as_float(v[u]), __uint_as_float(v[u + 1]));
                            const float2 e = __fadd2_rn(__ffma2_rn(s, make_float2(fb, fb), make_float2(ob, ob)), make_float2(-use, -use));
                            const float2 x = make_float2(ex2(e.x), ex2(e.y));
                            sum = __fadd2_rn(sum, x);
                            y[u / 2] = pack2(x.x, x.y);
                            if (PIECES == 2) {
                                const float2 z = unpack2(y[u / 2]);
                                y[8 + u / 2] = pack2(x.x - z.x, x.y - z.y);
                            }
                        }
                        L = fmaf(sum.x + sum.y, sh.rv[cs][b0 + b], L);
                        if (PIECES == 1)
                            tmem_st8(s_at + 8 * b, y);
                        else
                            tmem_st16(s_at + 16 * b, y);
                    });
                    // a scale that is not a number spoils the rows that see its block
                    for (unsigned bad = sh.poison[cs] >> b0 & 15u; bad; bad &= bad - 1)
                        if (seen > (__ffs(bad) - 1) * TQ_KV_BLOCK) L = __int_as_float(0x7fc00000);
                    tmem_wait_st();
                    tqp::tc_fence_before();
                    arrive(&sh.p_ready[t]);
                }
                together(); // the last w is read
                *put = L;
                together();
                L += *get;
                wait_slot(&sh.o_full[t], o_phase & 1, &sh.late, p.c.status);
                o_phase++;
                tqp::tc_fence_after();
            }
            // ---- out, or this part of it: some columns at a time through the rows' memory of Q, the halves apart ----
            const long long o_at_row = place(r, p.a.out_stride);
            constexpr int CH = PIECES * HDP / 16; // 16-byte chunks of a row there for a half
            auto staged = [&](int sr, int c) {    // chunk c of row sr of the warp
                const int ch = half * CH + c;
                return reinterpret_cast<uint4 *>(Qs + t * PIECES * OP + (ch >> 3) * (kRows * 128) +
                                                 chunk_at((warp & 3) * 32 + sr, ch & 7));
            };
            auto spread = [&](auto one, float factor, auto &&at) { // one: the element type
                using X = decltype(one);
                constexpr int E = 16 / sizeof(X), COLS = CH * E < OC ? CH * E : OC;
                constexpr int LANES = COLS / E, ROWS = 32 / LANES;
#pragma unroll 1
                for (int h = 0; h < OC; h += COLS) {
                    __syncwarp();
#pragma unroll 1
                    for (int c = 0; c < COLS; c += 16) {
                        uint32_t o[16];
                        tqp::tmem_ld16(o_at + h + c, o);
                        tqp::tmem_wait_ld();
#pragma unroll
                        for (int u = 0; u < 16; u += E) {
                            __align__(16) X e[E];
#pragma unroll
                            for (int k = 0; k < E; k += 2)
                                Elem<X>::put2(e + k, __uint_as_float(o[u + k]) * factor, __uint_as_float(o[u + k + 1]) * factor, true);
                            *staged(lane, (c + u) / E) = *reinterpret_cast<const uint4 *>(e);
                        }
                    }
                    __syncwarp();
                    const int c = lane % LANES;
#pragma unroll 1
                    for (int i = 0; i < 32; i += 4 * ROWS) {
                        uint4 x[4];
                        long long to[4];
#pragma unroll
                        for (int u = 0; u < 4; u++) {
                            const int sr = i + u * ROWS + lane / LANES;
                            x[u] = *staged(sr, c);
                            to[u] = __shfl_sync(0xffffffffu, o_at_row, sr);
                        }
#pragma unroll
                        for (int u = 0; u < 4; u++) at(i + u * ROWS + lane / LANES, half * OC + h + c * E, x[u], to[u]);
                    }
                }
                __syncwarp();
            };
            if (part_at < 0) {
                if (mine > 0)
                    spread(T(0.f), L == 0.f ? 0.f : 1.f / L, [&](int, int d, const uint4 &x, long long to) {
                        if (to < 0 || d >= p.c.hd) return;
                        T *o = static_cast<T *>(p.a.out) + to + d;
                        if (p.vec) {
                            *reinterpret_cast<uint4 *>(o) = x;
                        } else {
                            const T *e = reinterpret_cast<const T *>(&x);
#pragma unroll
                            for (int u = 0; u < 16 / (int)sizeof(T); u++) o[u] = e[u];
                        }
                    });
            } else {
                float *part = reinterpret_cast<float *>(static_cast<char *>(p.a.workspace) + kKvHead) +
                              ((size_t)blockIdx.x * 2 + part_at) * partial_floats(HDP);
                if (mine > 0)
                    spread(0.f, 1.f, [&](int sr, int d, const uint4 &x, long long) {
                        *reinterpret_cast<uint4 *>(part + (size_t)(t * kRows + (warp & 3) * 32 + sr) * HDP + d) = x;
                    });
                if (half == 0) {
                    const int pr = t * kRows + row;
                    part[kBlockRows * HDP + pr] = mine > 0 ? M : __int_as_float(0x7fc00000); // NaN: no part here
                    part[kBlockRows * HDP + kBlockRows + pr] = L;
                }
            }
            tick += cnt;
        }
    } else if (warp < kMmaWarp) {
        // ================= codes -> float16 operands =================
        const int ct = tid - 32 * kSoftWarps;
        constexpr int U = kPos * HDP / 16 / kConvThreads; // 16-byte words per thread and tile
        constexpr int PER_ROW = HDP / 16;
        static_assert(kPos * HDP / 16 == HDP * kBlocks, "a block is HDP words of 16 bytes");
        auto expand = [&](const uint4 &r, uint4 &lo, uint4 &hi) {
            cvt4(r.x, lo.x, lo.y);
            cvt4(r.y, lo.z, lo.w);
            cvt4(r.z, hi.x, hi.y);
            cvt4(r.w, hi.z, hi.w);
        };
        // a staged word, or zeros for a block that is not there
        auto word_of = [&](int side, int word, unsigned there) {
            const uint4 w = *reinterpret_cast<const uint4 *>(Cs + side * CODES + word * 16);
            return there >> (word / HDP) & 1 ? w : make_uint4(TQ_KV_BIAS, TQ_KV_BIAS, TQ_KV_BIAS, TQ_KV_BIAS);
        };
        unsigned k = 0;
        for (unsigned n = 0;; n++) {
            const int cnt = next_seg(n).cnt;
            __syncwarp();
            if (lane == 0) tqp::mbar_arrive(&sh.seg_empty[n % kSegs]);
            if (cnt == 0) break;
            for (const unsigned end = k + cnt; k < end; k++) {
                const unsigned s = k % ST, round = k / ST;
                // ---- keys ----
                wait_slot(&sh.code_full[0], k & 1, &sh.late, p.c.status);
                if (round > 0) wait_slot(&sh.k_empty[s], (round - 1) & 1, &sh.late, p.c.status);
                unsigned there = sh.live[0];
#pragma unroll 2
                for (int u = 0; u < U; u++) {
                    const int word = ct + u * kConvThreads, r = word / PER_ROW, c = word - r * PER_ROW;
                    // the word is stored at c: the 16 dimensions of chunk c ^ .. (tq_kv.h)
                    const int chunk = HDP >= 128 ? c ^ ((r & 1) << 2) : c;
                    uint4 a, b;
                    expand(word_of(0, word, there), a, b);
                    unsigned char *to = Ks + s * OP + (chunk >> 2) * (kPos * 128);
                    const int c0 = 2 * (chunk & 3), h = HDP >= 128 ? chunk >> 2 & 1 : 0; // halves in turn: distinct banks
                    *reinterpret_cast<uint4 *>(to + chunk_at(r, c0 + h)) = h ? b : a;
                    *reinterpret_cast<uint4 *>(to + chunk_at(r, c0 + 1 - h)) = h ? a : b;
                }
                tqp::fence_proxy_async();
                arrive(&sh.k_full[s]);
                if (lane == 0) tqp::mbar_arrive(&sh.code_empty[0]);
                // ---- values ----
                wait_slot(&sh.code_full[1], k & 1, &sh.late, p.c.status);
                if (round > 0) wait_slot(&sh.v_empty[s], (round - 1) & 1, &sh.late, p.c.status);
                there = sh.live[1];
#pragma unroll 2
                for (int u = 0; u < U; u++) {
                    const int word = ct + u * kConvThreads, blk = word / HDP, d = word - blk * HDP;
                    uint4 a, b;
                    expand(word_of(1, word, there), a, b);
                    unsigned char *to = Vs + s * OP + (blk >> 2) * (HDP * 128);
                    *reinterpret_cast<uint4 *>(to + chunk_at(d, 2 * (blk & 3))) = a;
                    *reinterpret_cast<uint4 *>(to + chunk_at(d, 2 * (blk & 3) + 1)) = b;
                }
                tqp::fence_proxy_async();
                arrive(&sh.v_full[s]);
                if (lane == 0) tqp::mbar_arrive(&sh.code_empty[1]);
            }
        }
    } else if (warp == kMmaWarp) {
        // ================= MMA issue: one thread =================
        if (lane == 0) {
            unsigned tick = 0, q_phase = 0, p_phase = 0; // phases: a bit for each row tile
            // descriptors differ in their address field alone: 16-byte units, no carry out of it
            const uint64_t dq = desc(tqp::smem_u32(Qs)), dk = desc(tqp::smem_u32(Ks)), dv = desc(tqp::smem_u32(Vs));
            auto scores = [&](auto t, unsigned n) { // S(t) = Q(t) K(n)^T
                const uint64_t kb = dk + (n % ST) * (OP >> 4);
#pragma unroll
                for (int pc = 0; pc < PIECES; pc++)
#pragma unroll
                    for (int ks = 0; ks < HDP / 16; ks++) {
                        const uint32_t o = ((ks >> 2) * (kRows * 128) + (ks & 3) * 32) >> 4;
                        mma_ss(s_col(t), dq + ((t * PIECES + pc) * (OP >> 4) + o), kb + o, idesc_f16(kPos), pc > 0 || ks > 0);
                    }
                tqp::umma_commit(&sh.s_full[t]);
            };
            auto products = [&](auto t, unsigned n, bool first) { // O(t) += P(t) V(n)
                const uint64_t vb = dv + (n % ST) * (OP >> 4);
#pragma unroll
                for (int pc = 0; pc < PIECES; pc++)
#pragma unroll
                    for (int ks = 0; ks < kPos / 16; ks++) {
                        const uint32_t a = // a half's blocks lie behind one another (two pieces: side by side)
                            PIECES == 1 ? s_col(t) + (ks >> 2) * (kPos / 2) + 8 * (ks & 3) : s_col(t) + 16 * ks + 8 * pc;
                        mma_ts(o_col(t), a, vb + (((ks >> 2) * (HDP * 128) + (ks & 3) * 32) >> 4), idesc_f16(HDP),
                               pc > 0 || ks > 0 ? 1u : !first);
                    }
            };
            auto wait_tile = [&](uint64_t *bars, auto t, unsigned &phase) {
                wait_slot(&bars[t], phase >> t & 1, &sh.late, p.c.status);
                phase ^= 1u << t;
            };
            for (unsigned sn = 0;; sn++) {
                const Seg &g = next_seg(sn);
                const int cnt = g.cnt, mine_a = g.mine[0], mine_b = g.mine[1];
                tqp::mbar_arrive(&sh.seg_empty[sn % kSegs]);
                if (cnt == 0) break;
                for (int j = -1; j < cnt; j++) {
                    const unsigned n = tick + j;
                    // every tile's operands are waited for once, whether a row tile uses them or not
                    auto half_step = [&](auto t, int mine) {
                        if (j >= 0 && t == 0) wait_slot(&sh.v_full[n % ST], (n / ST) & 1, &sh.late, p.c.status);
                        if (j >= 0 && j < mine) {
                            wait_tile(sh.p_ready, t, p_phase);
                            tqp::tc_fence_after();
                            products(t, n, j == 0);
                            if (j + 1 == mine) tqp::umma_commit(&sh.o_full[t]);
                        }
                        if (j >= 0 && t == 1) tqp::umma_commit(&sh.v_empty[n % ST]);
                        if (j + 1 < cnt && t == 0)
                            wait_slot(&sh.k_full[(n + 1) % ST], ((n + 1) / ST) & 1, &sh.late, p.c.status);
                        if (j + 1 < mine) {
                            if (j < 0) wait_tile(sh.q_ready, t, q_phase);
                            tqp::tc_fence_after();
                            scores(t, n + 1);
                        }
                        if (j + 1 < cnt && t == 1) tqp::umma_commit(&sh.k_empty[(n + 1) % ST]);
                    };
                    half_step(std::integral_constant<int, 0>(), mine_a);
                    half_step(std::integral_constant<int, 1>(), mine_b);
                }
                tick += cnt;
            }
        }
    } else {
        // ================= loader: segments, pages, codes =================
        const TqSplit split(total, G);
        const long long x0 = split.start(blockIdx.x), x1 = split.start(blockIdx.x + 1);
        const float mag = fabsf(p.scale2);
        // Lanes 0..7 take a block of the tile each. A tile passes through three
        // stages: its page is asked for, then its scales, then its codes; the
        // first runs two tiles ahead of the last, across segments.
        Where w = find(p, sums, x0);
        __syncwarp(); // the sums are read: codes go over them
        int tile = 0, left = 0, visible = 0; // of the first stage
        unsigned n = 0;
        const int *table = nullptr;
        // Hands the segment at w, or the next that has position tiles here, to the
        // other roles; without one, the end.
        auto open = [&]() {
            for (;; next_segment(p, w)) {
                left = 0;
                if (w.i >= p.a.n || w.from - kSegCost >= x1) break;
                tile = w.first(x0);
                left = w.first(x1) - tile;
                if (left > 0) break;
            }
            if (n >= kSegs) wait_slot(&sh.seg_empty[n % kSegs], (n / kSegs - 1) & 1, &sh.late, p.c.status);
            if (lane == 0) {
                Seg &g = sh.seg[n % kSegs];
                g.cnt = left;
                if (left > 0) {
                    g.start = w.s.start, g.nq = w.s.nq, g.len = w.s.len;
                    g.head = w.head, g.row0 = w.rb * kBlockRows;
                    g.tile = tile;
                    for (int t = 0; t < 2; t++) g.mine[t] = min(left, max(0, tiles_of(w, t, group) - tile));
                    g.part = left == w.tiles ? -1 : tile == 0 ? 1 : 0;
                }
                tqp::mbar_arrive(&sh.seg_full[n % kSegs]);
            }
            n++;
            if (left == 0) return;
            visible = sees(w.s, min(w.s.nq * group, (w.rb + 1) * kBlockRows) - 1, group);
            table = p.a.table + (size_t)w.i * p.a.table_stride;
        };
        struct Block {
            int id, head, in;  // page, KV head, block of the page; id < 0: not there
            bool wanted, some; // some: there is such a tile
        };
        auto ask_page = [&]() { // first stage: the next tile
            Block b{-1, 0, 0, false, false};
            if (left == 0) return b;
            const int pos = tile * kPos + lane * TQ_KV_BLOCK;
            b.head = w.head;
            b.in = (pos & (p.c.page - 1)) >> 4;
            b.wanted = lane < kBlocks && pos < visible;
            if (b.wanted) b.id = __ldg(table + (pos >> p.c.page_shift));
            b.some = true;
            tile++;
            if (--left == 0) {
                next_segment(p, w);
                open();
            }
            return b;
        };
        auto ask_scales = [&](Block &b) { // second stage
            if (b.wanted && (b.id < 0 || b.id >= p.c.n_pages)) {
                atomicOr(p.c.status, TQ_KV_STATUS_PAGE);
                b.id = -1;
            }
            return b.id >= 0 ? __ldg(p.c.scale + (size_t)b.id * p.c.n_kv + b.head) : make_float2(0.f, 0.f);
        };
        open();
        Block b0 = ask_page(), b1 = ask_page();
        float2 sc = ask_scales(b0);
        for (unsigned k = 0; b0.some; k++) {
            const Block b2 = ask_page();
            const float2 sc1 = ask_scales(b1);
            const bool there = b0.id >= 0, some = there && !(sc.y < kLeastValue);
            const size_t at = there ? kv_block_offset(p.c, b0.id, b0.head, b0.in) : 0;
            const unsigned keys = __ballot_sync(0xffffffffu, there), values = __ballot_sync(0xffffffffu, some);
            const unsigned nan = __ballot_sync(0xffffffffu, there && (sc.x != sc.x || sc.y != sc.y));
            // ---- keys, and the scales ----
            if (k > 0) wait_slot(&sh.code_empty[0], (k - 1) & 1, &sh.late, p.c.status);
            if (lane < kBlocks) {
                const bool use = there && !(nan >> lane & 1), plain = use && sc.y >= kLeastValue;
                sh.f[k % kConsts][lane] = use ? sc.x * mag : 0.f;
                sh.lv[k % kConsts][lane] = !use ? -INFINITY : log2f(plain ? sc.y : kNoValue);
                sh.rv[k % kConsts][lane] = !use ? 0.f : 1.f / (plain ? sc.y : kNoValue);
            }
            if (lane == 0) sh.live[0] = keys, sh.poison[k % kConsts] = nan;
            __syncwarp();
            if (lane == 0) tqp::mbar_arrive_expect_tx(&sh.code_full[0], __popc(keys) * TQ_KV_BLOCK * HDP);
            __syncwarp();
            if (there) tqp::bulk_load(Cs + lane * TQ_KV_BLOCK * HDP, p.c.k + at, TQ_KV_BLOCK * HDP, &sh.code_full[0]);
            // ---- values ----
            if (k > 0) wait_slot(&sh.code_empty[1], (k - 1) & 1, &sh.late, p.c.status);
            if (lane == 0) {
                sh.live[1] = values;
                tqp::mbar_arrive_expect_tx(&sh.code_full[1], __popc(values) * TQ_KV_BLOCK * HDP);
            }
            __syncwarp();
            if (some)
                tqp::bulk_load(Cs + CODES + lane * TQ_KV_BLOCK * HDP, p.c.v + at, TQ_KV_BLOCK * HDP, &sh.code_full[1]);
            b0 = b1, b1 = b2, sc = sc1;
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
    __shared__ long long sums[kKvSums + 1], scan[kJoinThreads / 32];
    const long long total = list_sums<kJoinThreads>(p, sums, scan);
    const int G = (int)min((long long)grid, (total + kMinUnits - 1) / kMinUnits);
    const int cta = blockIdx.x;
    if (cta + 1 >= G) return;
    const TqSplit split(total, G);
    const long long c0 = split.start(cta), c1 = split.start(cta + 1);
    const Where w = find(p, sums, c1 - 1);
    // its position tiles begin here and end elsewhere?
    if (w.from < c0 || w.from >= c1 || w.from + w.tiles <= c1) return;
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
        Elem<T>::put2(o, A.x * inv, A.y * inv, p.vec);
        Elem<T>::put2(o + 2, A.z * inv, A.w * inv, p.vec);
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
