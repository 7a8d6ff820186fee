// tq_kv_attn.cu — attention over the paged 8-bit cache (tq_kv_attention_dev;
// layout in tq_kv.h).
//
// For a query row q and the positions t that it sees, with codes k_t, v_t and
// the scales a_b, c_b of the block b that holds t:
//   s_t = (q . k_t) a_b scale log2(e),  m = max s_t,  p_t = 2^(s_t - m),
//   out = sum_t p_t c_b v_t / sum_t p_t,
// in one pass over the positions with a running m, sum and accumulator.
//
// Rows. The query heads of a KV head, for all new tokens of a sequence, are the
// rows of one product, in tiles of R = 16 / PIECES rows of an m16n8k16 MMA.
// Codes are exact in float16. With PIECES = 2 a row takes two MMA rows, q = hi
// + lo (and p likewise), each a float16, which keeps 22 bits of both: float32
// products for float32 queries, at no cost while a KV head has at most 8 rows.
// With PIECES = 1 a 16-bit q is one float16 (exact: the row is scaled by a power
// of two first) and p is rounded to 11 bits, below the output's own rounding.
// c_b rides on p: p_t c_b / C with C the largest c_b so far (a running value
// like m), so that it stays in float16's range; the sum of p itself is float32.
//
// Work. A warp takes 64 positions at a time: keys and values come by bulk copies
// of 16-position blocks into its own ring of three slots (k, v, k, ..), two of
// them in flight while one is used, and go from there straight into MMA
// fragments: sixteen dimensions of a key, or sixteen positions of a value
// dimension, are one 16-byte read, and q and p are permuted to match. The scores
// of the MMA's accumulator are the next product's operand in place.
// All (sequence, KV head, row tile) segments laid end to end are cut evenly over
// the CTAs, then over their warps, wherever the cuts fall (lengths are device
// data; every CTA makes the same sums). A warp's unfinished segments meet in its
// CTA, the CTA's in the CTA that arrives last, in a fixed order: results do not
// depend on timing.
#include <climits>

#include "tq_kv_attn.cuh"

namespace {

using namespace tqkv;
using Params = TqKvParams;

constexpr int kTile = 64;       // positions per step of a warp
constexpr int kSlots = 3;       // ring slots per warp
constexpr int kWide = 4;        // MMA accumulators worked on in turn
constexpr int kMinTiles = 4;    // tiles per CTA below which fewer CTAs work
constexpr int kPromptRows = 48; // rows of a sequence above which the prompt kernel takes it
constexpr int kDirect = 1024;   // sequences whose lengths are kept in shared memory
constexpr int kSums = kKvSums;
constexpr float kPUnit = 16384.f; // p = 1 in float16: its low piece stays normal
constexpr size_t kHead = kKvHead;
constexpr int kMaxGrid = kHead / sizeof(unsigned);

constexpr int warps_of(int hdp) { return hdp == 256 ? 4 : 8; }
constexpr int ctas_of(int hdp) { return hdp == 64 ? 2 : 1; } // CTAs per SM
constexpr int slot_bytes(int hdp) { return kTile * hdp + 128; }
constexpr int value_pitch(int hdp) { return TQ_KV_BLOCK * hdp + 32; } // four blocks in distinct banks
constexpr int partial_floats(int hdp) { return 16 * (hdp + 2); }
constexpr int partials_of(int hdp) { return 2 * warps_of(hdp) + 2; } // per CTA
constexpr size_t smem_bytes(int hdp) {
    return (size_t)warps_of(hdp) * kSlots * slot_bytes(hdp) + sizeof(long long) * (kSums + 1) +
           sizeof(int) * (2 * kDirect + 2);
}

template <int HDP, int PIECES, typename T>
__global__ void __launch_bounds__(32 * warps_of(HDP), ctas_of(HDP)) kv_attn_kernel(const __grid_constant__ Params p) {
    constexpr int NW = warps_of(HDP), NT = 32 * NW, R = 16 / PIECES, KK = HDP / 64, NI = HDP / 8;
    extern __shared__ __align__(128) unsigned char sm[];
    long long *sums = reinterpret_cast<long long *>(sm + (size_t)NW * kSlots * slot_bytes(HDP));
    int *s_starts = reinterpret_cast<int *>(sums + kSums + 1), *s_lens = s_starts + kDirect + 1;
    __shared__ uint64_t bars[NW][kSlots];
    __shared__ long long s_scan[NW + 1];
    __shared__ long long e_seg[2 * NW], e_end[2 * NW]; // unfinished segments of the warps: first and last tile + 1
    __shared__ int e_row[2 * NW][3];                   // their sequence, KV head, row tile
    __shared__ volatile int s_late;
    __shared__ int s_last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int n = p.a.n, n_kv = p.c.n_kv, group = p.group;

    // ---- lengths, checked; sums of the sequences' tiles --------------------------------
    const bool direct = n <= kDirect;
    if (direct) {
        for (int i = tid; i <= n; i += NT) s_starts[i] = p.a.starts[i];
        for (int i = tid; i < n; i += NT) s_lens[i] = p.a.lens[i];
    }
    if (lane < kSlots) tqp::mbar_init(&bars[warp][lane], 1);
    if (tid == 0) s_late = 0;
    if (tid < 2 * NW) e_seg[tid] = -1;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncthreads();
    const int *starts = direct ? s_starts : p.a.starts, *lens = direct ? s_lens : p.a.lens;
    auto seq_of = [&](int i) {
        Seq s = seq_at(p, starts, lens, i);
        if (s.nq > p.rows_cut / group) s.nq = 0; // the prompt kernel's
        return s;
    };
    auto tiles_per = [](const Seq &s) { return s.len > kTile ? (s.len + kTile - 1) / kTile : 1; };
    auto row_tiles = [&](const Seq &s) { return (s.nq * group + R - 1) / R; };
    const int span = 1 << p.shift_sums, entries = (n + span - 1) >> p.shift_sums;
    long long total;
    { // kSums entries over NT threads
        constexpr int PER = kSums / NT;
        long long own[PER], sum = 0;
#pragma unroll
        for (int u = 0; u < PER; u++) {
            const int e = tid * PER + u;
            own[u] = 0;
            for (int i = e << p.shift_sums; e < entries && i < min(n, (e + 1) << p.shift_sums); i++) {
                const Seq s = seq_of(i);
                own[u] += (long long)row_tiles(s) * n_kv * tiles_per(s);
            }
            sum += own[u];
        }
        long long inc = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        if (lane == 31) s_scan[warp] = inc;
        __syncthreads();
        long long before = 0;
        total = 0;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            if (w < warp) before += s_scan[w];
            total += s_scan[w];
        }
        before += inc - sum;
#pragma unroll
        for (int u = 0; u < PER; u++) {
            const int e = tid * PER + u;
            if (e <= entries) sums[e] = before;
            before += own[u];
        }
        if (tid == 0 && entries == kSums) sums[kSums] = total;
        __syncthreads();
    }
    // ---- this CTA's and this warp's tiles ------------------------------------------------
    const int G = (int)min((long long)gridDim.x, max(1ll, (total + kMinTiles - 1) / kMinTiles));
    if ((int)blockIdx.x >= G || total == 0) return;
    const TqSplit split(total, G);
    const long long c0 = split.start(blockIdx.x), c1 = split.start(blockIdx.x + 1);
    const long long x0 = c0 + (c1 - c0) * warp / NW, x1 = c0 + (c1 - c0) * (warp + 1) / NW;
    float *part = reinterpret_cast<float *>(static_cast<char *>(p.a.workspace) + kHead);
    auto partial_at = [&](int cta, int k) { return part + ((size_t)cta * partials_of(HDP) + k) * partial_floats(HDP); };

    struct Cursor {
        int i, seg, tile, tps, nrt, nseg;
        Seq s;
    };
    auto enter = [&](Cursor &c) { // a sequence's figures
        c.s = seq_of(c.i);
        c.tps = tiles_per(c.s);
        c.nrt = row_tiles(c.s);
        c.nseg = c.nrt * n_kv;
    };
    auto advance = [&](Cursor &c) {
        if (++c.tile < c.tps) return;
        c.tile = 0;
        if (++c.seg < c.nseg) return;
        c.seg = 0;
        do {
            c.i++;
            if (c.i >= n) return;
            enter(c);
        } while (c.nseg == 0);
    };
    // positions that some row of the cursor's segment sees
    auto seen_by = [&](const Cursor &c) {
        const int rt = c.seg % c.nrt, last = min((rt + 1) * R, c.s.nq * group) - 1;
        return min(c.s.len, max(0, c.s.len - c.s.nq + last / group + 1));
    };

    unsigned char *ring = sm + (size_t)warp * kSlots * slot_bytes(HDP);
    if (x0 < x1) {
        Cursor cur;
        {
            int lo = 0, hi = entries;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (sums[mid] <= x0)
                    lo = mid;
                else
                    hi = mid;
            }
            long long rest = x0 - sums[lo];
            cur.i = lo << p.shift_sums;
            enter(cur);
            while (rest >= (long long)cur.nseg * cur.tps) {
                rest -= (long long)cur.nseg * cur.tps;
                cur.i++;
                enter(cur);
            }
            cur.seg = (int)(rest / cur.tps);
            cur.tile = (int)(rest - (long long)cur.seg * cur.tps);
        }
        // ---- the loader: one tile's keys, then its values; item = 2 * tile number + (0 | 1) --
        Cursor ld = cur;
        long long left = x1 - x0; // tiles still to be loaded
        int nid = -1, vid = -1, n_head = 0, v_head = 0;
        unsigned item = 0;
        auto fetch_id = [&]() { // the page of this lane's block (t) of the loader's tile
            nid = -1;
            if (left <= 0) return;
            const int pos = ld.tile * kTile + t * TQ_KV_BLOCK;
            n_head = ld.seg / ld.nrt;
            if (pos < seen_by(ld)) {
                nid = p.a.table[(size_t)ld.i * p.a.table_stride + (pos >> p.c.page_shift)];
                if (nid < 0 || nid >= p.c.n_pages) {
                    nid = -1;
                    atomicOr(p.c.status, TQ_KV_STATUS_PAGE);
                }
            }
        };
        auto copy = [&](const int8_t *from, int id, int head, int in_page, int pitch) {
            const unsigned slot = item % kSlots;
            unsigned char *to = ring + slot * slot_bytes(HDP);
            const int blocks = __popc(__ballot_sync(0xffffffffu, id >= 0) & 15u);
            if (lane == 0) tqp::mbar_arrive_expect_tx(&bars[warp][slot], blocks * TQ_KV_BLOCK * HDP);
            __syncwarp();
            if (lane < 4 && id >= 0)
                tqp::bulk_load(to + lane * pitch, from + kv_block_offset(p.c, id, head, in_page), TQ_KV_BLOCK * HDP,
                               &bars[warp][slot]);
            item++;
        };
        int n_block = 0, v_block = 0;
        auto load_keys = [&](float2 &sc) { // and this lane's block's scales; x < 0: a block that is not there
            sc = make_float2(-1.f, 0.f);
            if (left <= 0) return;
            n_block = ((ld.tile * kTile + t * TQ_KV_BLOCK) & (p.c.page - 1)) >> 4;
            copy(p.c.k, nid, n_head, n_block, TQ_KV_BLOCK * HDP);
            if (nid >= 0) sc = __ldg(p.c.scale + (size_t)nid * n_kv + n_head);
            vid = nid, v_head = n_head, v_block = n_block;
            left--;
            if (left > 0) advance(ld);
            fetch_id();
        };
        auto load_values = [&]() { copy(p.c.v, vid, v_head, v_block, value_pitch(HDP)); };

        float2 sc, sc_next;
        fetch_id();
        load_keys(sc);
        load_values();
        load_keys(sc_next);
        unsigned used = 0; // items used

        unsigned qf[KK][4][4];
        float O[NI][4];
        float m[2], l[2], C = 0.f, row_unit[2];
        int lim[2], least = 0;
        bool fresh = true;
        long long seg_from = 0;
        const long long ntile = x1 - x0;
        for (long long x = 0; x < ntile; x++) {
            const int head = cur.seg / cur.nrt, rt = cur.seg - head * cur.nrt;
            if (fresh) {
                fresh = false;
                seg_from = x0 + x - cur.tile;
                const int rows = cur.s.nq * group;
                least = cur.s.len;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    m[h] = -INFINITY;
                    l[h] = 0.f;
                    row_unit[h] = 1.f;
                    lim[h] = cur.s.len;
                }
                C = 0.f;
#pragma unroll
                for (int i = 0; i < NI; i++) O[i][0] = O[i][1] = O[i][2] = O[i][3] = 0.f;
                least = min(cur.s.len, max(0, cur.s.len - cur.s.nq + rt * R / group + 1));
#pragma unroll
                for (int h = 0; h < 3 - PIECES; h++) { // MMA rows g and, with one piece, g + 8
                    const int row = rt * R + g + 8 * h;
                    const int tok = row / group, hq = head * group + row - tok * group;
                    const bool live = row < rows;
                    float x[KK][16];
                    float big = 0.f;
                    const T *q = static_cast<const T *>(p.a.q) + (size_t)(cur.s.start + tok) * p.a.q_stride +
                                 (size_t)hq * p.c.hd;
#pragma unroll
                    for (int kk = 0; kk < KK; kk++)
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            const int d = 64 * kk + 16 * t + 8 * j;
                            float y[8];
                            if (live && d < p.c.hd)
                                load8(q + d, p.vec, y);
                            else
#pragma unroll
                                for (int u = 0; u < 8; u++) y[u] = 0.f;
#pragma unroll
                            for (int u = 0; u < 8; u++) {
                                x[kk][8 * j + u] = y[u];
                                big = fmaxf(big, fabsf(y[u]));
                            }
                        }
                    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
                    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
                    const float unit = row_scale(big, &row_unit[h]);
                    if (live) lim[h] = min(cur.s.len, max(0, cur.s.len - cur.s.nq + tok + 1));
#pragma unroll
                    for (int kk = 0; kk < KK; kk++)
#pragma unroll
                        for (int u = 0; u < 4; u++)
#pragma unroll
                            for (int e = 0; e < 2; e++) { // dimensions 4u + 2e, + 1 of the lane's sixteen
                                const float y0 = x[kk][4 * u + 2 * e] * unit, y1 = x[kk][4 * u + 2 * e + 1] * unit;
                                const unsigned hi = pack2(y0, y1);
                                qf[kk][u][2 * e + h] = hi;
                                if (PIECES == 2) {
                                    const float2 b = unpack2(hi);
                                    qf[kk][u][2 * e + 1] = pack2(y0 - b.x, y1 - b.y);
                                }
                            }
                }
                if (PIECES == 2) lim[1] = lim[0];
            }
            // ---- s = q . k for 64 positions ----
            const int pos0 = cur.tile * kTile;
            float S[8][4];
#pragma unroll
            for (int j = 0; j < 8; j++) S[j][0] = S[j][1] = S[j][2] = S[j][3] = 0.f;
            wait_slot(&bars[warp][used % kSlots], (used / kSlots) & 1, &s_late, p.c.status);
            {
                const unsigned char *ks = ring + (used % kSlots) * slot_bytes(HDP) + (g >> 1) * TQ_KV_BLOCK * HDP +
                                          (g & 1) * HDP;
#pragma unroll
                for (int kk = 0; kk < KK; kk++) {
                    const int ch = HDP >= 128 ? (4 * kk + t) ^ ((g & 1) << 2) : 4 * kk + t;
#pragma unroll
                    for (int j0 = 0; j0 < 8; j0 += kWide) { // kWide sums in turn: none waits for its last product
                        uint4 w[kWide];
#pragma unroll
                        for (int j = 0; j < kWide; j++)
                            w[j] = *reinterpret_cast<const uint4 *>(ks + (j0 + j) * 2 * HDP + ch * 16);
#pragma unroll
                        for (int u = 0; u < 4; u++)
#pragma unroll
                            for (int j = 0; j < kWide; j++) {
                                unsigned b0, b1;
                                cvt4((&w[j].x)[u], b0, b1);
                                mma16816(S[j0 + j], qf[kk][u], b0, b1);
                            }
                    }
                }
            }
            used++;
            __syncwarp(); // the slot is read
            if (x + 1 < ntile) load_values();
            // ---- softmax of the lane's 16 positions (its block), per row ----
            const bool there = sc.x >= 0.f || sc.x != sc.x;
            const bool whole = pos0 + kTile <= least && __all_sync(0xffffffffu, there);
            const float a = there ? sc.x * p.scale2 : 0.f;
            float cmax = there ? sc.y : 0.f;
            cmax = fmaxf(cmax, __shfl_xor_sync(0xffffffffu, cmax, 1));
            cmax = fmaxf(cmax, __shfl_xor_sync(0xffffffffu, cmax, 2));
            const float C1 = fmaxf(C, cmax);
            const float keepC = C1 > 0.f ? C / C1 : 1.f;
            const float ride = C1 > 0.f ? (there ? sc.y : 0.f) / C1 * kPUnit : (there ? sc.y : 0.f);
            C = C1;
            constexpr int H = 3 - PIECES;
            float alpha[2];
            unsigned pf[4][4];
#pragma unroll
            for (int h = 0; h < H; h++) {
                const float f = a * row_unit[h];
                float v[16], mx = -INFINITY;
                unsigned hidden = 0; // positions that the row does not see: p = 0 whatever their scales are
#pragma unroll
                for (int j = 0; j < 8; j++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float s = PIECES == 2 ? S[j][e] + S[j][2 + e] : S[j][2 * h + e];
                        s *= f;
                        if (!whole && (!there || pos0 + 16 * t + 2 * j + e >= lim[h])) {
                            s = -INFINITY;
                            hidden |= 1u << (2 * j + e);
                        }
                        v[2 * j + e] = s;
                        mx = fmaxf(mx, s);
                    }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float m1 = fmaxf(m[h], mx), base = m1 == -INFINITY ? 0.f : m1;
                const float up = exp2f(m[h] - base);
                alpha[h] = up * keepC;
                m[h] = m1;
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    v[j] = exp2f(v[j] - base);
                    sum += v[j];
                    v[j] = !whole && (hidden >> j & 1) ? 0.f : v[j] * ride;
                }
                l[h] = l[h] * up + sum;
#pragma unroll
                for (int u = 0; u < 4; u++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const unsigned hi = pack2(v[4 * u + 2 * e], v[4 * u + 2 * e + 1]);
                        pf[u][2 * e + h] = hi;
                        if (PIECES == 2) {
                            const float2 b = unpack2(hi);
                            pf[u][2 * e + 1] = pack2(v[4 * u + 2 * e] - b.x, v[4 * u + 2 * e + 1] - b.y);
                        }
                    }
            }
            if (PIECES == 2) alpha[1] = alpha[0];
            if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
                for (int i = 0; i < NI; i++) {
                    O[i][0] *= alpha[0];
                    O[i][1] *= alpha[0];
                    O[i][2] *= alpha[1];
                    O[i][3] *= alpha[1];
                }
            }
            // ---- O += p v ----
            wait_slot(&bars[warp][used % kSlots], (used / kSlots) & 1, &s_late, p.c.status);
            {
                const unsigned char *vs = ring + (used % kSlots) * slot_bytes(HDP) + t * value_pitch(HDP) + g * 16;
#pragma unroll
                for (int i0 = 0; i0 < NI; i0 += kWide) {
                    uint4 w[kWide];
#pragma unroll
                    for (int i = 0; i < kWide; i++) w[i] = *reinterpret_cast<const uint4 *>(vs + (i0 + i) * 128);
#pragma unroll
                    for (int u = 0; u < 4; u++)
#pragma unroll
                        for (int i = 0; i < kWide; i++) {
                            unsigned b0, b1;
                            cvt4((&w[i].x)[u], b0, b1);
                            mma16816(O[i0 + i], pf[u], b0, b1);
                        }
                }
            }
            used++;
            __syncwarp();
            sc = sc_next;
            load_keys(sc_next);
            // ---- the segment's end, or the warp's ----
            const bool ends = cur.tile + 1 == cur.tps;
            if (ends || x + 1 == ntile) {
                const float unit = C / kPUnit;
#pragma unroll
                for (int h = 0; h < H; h++) {
                    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
                    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
                }
                const bool began = seg_from >= x0;
                const int rows = cur.s.nq * group;
                if (ends && began) {
#pragma unroll
                    for (int h = 0; h < H; h++) {
                        const int row = rt * R + g + 8 * h;
                        if (row >= rows) continue;
                        const int tok = row / group, hq = head * group + row - tok * group;
                        T *o = static_cast<T *>(p.a.out) + (size_t)(cur.s.start + tok) * p.a.out_stride +
                               (size_t)hq * p.c.hd;
                        const float inv = l[h] == 0.f ? 0.f : unit / l[h];
#pragma unroll
                        for (int i = 0; i < NI; i++) {
                            const int d = 8 * i + 2 * t;
                            const float y0 = PIECES == 2 ? O[i][0] + O[i][2] : O[i][2 * h];
                            const float y1 = PIECES == 2 ? O[i][1] + O[i][3] : O[i][2 * h + 1];
                            if (d < p.c.hd) Elem<T>::put2(o + d, y0 * inv, y1 * inv, p.vec, true);
                        }
                    }
                } else { // to be joined: sums in plain units, m and l
                    const int k = began ? 1 : 0, e = 2 * warp + k;
                    float *to = partial_at(blockIdx.x, e);
#pragma unroll
                    for (int h = 0; h < H; h++) {
#pragma unroll
                        for (int i = 0; i < NI; i++) {
                            const float y0 = PIECES == 2 ? O[i][0] + O[i][2] : O[i][2 * h];
                            const float y1 = PIECES == 2 ? O[i][1] + O[i][3] : O[i][2 * h + 1];
                            *reinterpret_cast<float2 *>(to + (g + 8 * h) * HDP + 8 * i + 2 * t) =
                                make_float2(y0 * unit, y1 * unit);
                        }
                        if (t == 0) {
                            to[16 * HDP + g + 8 * h] = m[h];
                            to[16 * HDP + 16 + g + 8 * h] = l[h];
                        }
                    }
                    if (lane == 0) {
                        e_seg[e] = seg_from;
                        e_end[e] = seg_from + cur.tps;
                        e_row[e][0] = cur.i;
                        e_row[e][1] = head;
                        e_row[e][2] = rt;
                    }
                }
                fresh = true;
            }
            if (x + 1 < ntile) advance(cur);
        }
    }
    __syncthreads();

    // ---- join the warps' unfinished segments, then the CTAs' ------------------------------
    // Sum of the partials `at(0..k)`; thread: 4 dimensions of a row at a time.
    auto join = [&](auto at, int k, int i, int head, int rt, float *to) {
        const Seq s = seq_of(i);
        const int rows = min(R, s.nq * group - rt * R);
        for (int e = tid; e < rows * (HDP / 4); e += NT) {
            const int r = e / (HDP / 4), d = (e - r * (HDP / 4)) * 4;
            float M = -INFINITY;
            for (int j = 0; j < k; j++) M = fmaxf(M, __ldcg(at(j) + 16 * HDP + r));
            const float base = M == -INFINITY ? 0.f : M;
            float L = 0.f;
            float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int j = 0; j < k; j++) {
                const float *f = at(j);
                const float w = exp2f(__ldcg(f + 16 * HDP + r) - base);
                const float4 y = __ldcg(reinterpret_cast<const float4 *>(f + r * HDP + d));
                L += w * __ldcg(f + 16 * HDP + 16 + r);
                A.x += w * y.x;
                A.y += w * y.y;
                A.z += w * y.z;
                A.w += w * y.w;
            }
            if (to) {
                *reinterpret_cast<float4 *>(to + r * HDP + d) = A;
                if (d == 0) to[16 * HDP + r] = M, to[16 * HDP + 16 + r] = L;
            } else if (d < p.c.hd) {
                const int row = rt * R + r, tok = row / group, hq = head * group + row - tok * group;
                T *o = static_cast<T *>(p.a.out) + (size_t)(s.start + tok) * p.a.out_stride + (size_t)hq * p.c.hd + d;
                const float inv = L == 0.f ? 0.f : 1.f / L;
                Elem<T>::put2(o, A.x * inv, A.y * inv, p.vec, true);
                Elem<T>::put2(o + 2, A.z * inv, A.w * inv, p.vec, true);
            }
        }
    };
    unsigned *counters = static_cast<unsigned *>(p.a.workspace);
    for (int e = 0; e < 2 * NW;) {
        const long long seg = e_seg[e];
        if (seg < 0) {
            e++;
            continue;
        }
        // the run of partials of this segment (empty places between them are skipped)
        int list[2 * NW], k = 0, f = e;
        for (; f < 2 * NW; f++) {
            if (e_seg[f] < 0) continue;
            if (e_seg[f] != seg) break;
            list[k++] = f;
        }
        const long long end = e_end[e];
        const int i = e_row[e][0], head = e_row[e][1], rt = e_row[e][2];
        auto mine = [&](int j) -> const float * { return partial_at(blockIdx.x, list[j]); };
        if (seg >= c0 && end <= c1) {
            join(mine, k, i, head, rt, nullptr);
        } else {
            const int first = split.owner(seg), last = split.owner(end - 1);
            join(mine, k, i, head, rt, partial_at(blockIdx.x, 2 * NW + ((int)blockIdx.x == first ? 1 : 0)));
            __syncthreads();
            if (tid == 0) s_last = tq_arrive_last(counters + first, last - first + 1);
            __syncthreads();
            if (s_last)
                join([&](int j) -> const float * { return partial_at(first + j, 2 * NW + (j == 0 ? 1 : 0)); },
                     last - first + 1, i, head, rt, nullptr);
        }
        e = f;
    }
}

template <int HDP, int PIECES, typename T>
cudaError_t launch(const Params &p, int sms, cudaStream_t st) {
    static TqDeviceOnce once;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess)
        e = tq_device_once(once, dev, [] {
            return cudaFuncSetAttribute(kv_attn_kernel<HDP, PIECES, T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        (int)smem_bytes(HDP));
        });
    if (e != cudaSuccess) return e;
    const int grid = min(kMaxGrid, sms * ctas_of(HDP));
    kv_attn_kernel<HDP, PIECES, T><<<grid, 32 * warps_of(HDP), smem_bytes(HDP), st>>>(p);
    return cudaGetLastError();
}

template <int HDP> cudaError_t launch_hd(const Params &p, int sms, cudaStream_t st) {
    // Two pieces keep float32's precision; a 16-bit query takes one piece when its
    // rows of one token would not fit the eight that two pieces leave.
    const bool two = p.a.dtype == TQ_LINEAR_F32 || p.group <= 8;
    if (p.a.dtype == TQ_LINEAR_F32) return launch<HDP, 2, float>(p, sms, st);
    if (p.a.dtype == TQ_LINEAR_F16) return two ? launch<HDP, 2, __half>(p, sms, st) : launch<HDP, 1, __half>(p, sms, st);
    return two ? launch<HDP, 2, __nv_bfloat16>(p, sms, st) : launch<HDP, 1, __nv_bfloat16>(p, sms, st);
}

} // namespace

static size_t small_workspace(int hdp, int sms) {
    const size_t grid = (size_t)(sms * ctas_of(hdp) < kMaxGrid ? sms * ctas_of(hdp) : kMaxGrid);
    return kHead + grid * partials_of(hdp) * partial_floats(hdp) * sizeof(float);
}
size_t tq_kv_attn_workspace(int hdp, int sms) {
    const size_t a = small_workspace(hdp, sms), b = tq_kv_prompt_workspace(hdp, sms);
    return a > b ? a : b; // the two kernels of a call run one after the other
}

cudaError_t tq_kv_launch_attn(const TqKvView &v, const TqKvAttn &a, int sms, cudaStream_t st) {
    Params p;
    p.c = v;
    p.a = a;
    p.group = a.n_q / v.n_kv;
    const size_t es = a.dtype == TQ_LINEAR_F32 ? 4 : 2;
    const size_t bits = (uintptr_t)a.q | (uintptr_t)a.out | (size_t)(a.q_stride * (long long)es) |
                        (size_t)(a.out_stride * (long long)es) | (size_t)v.hd * es;
    p.vec = bits % 16 == 0;
    p.shift_sums = 0;
    while ((a.n >> p.shift_sums) > kSums - 1) p.shift_sums++;
    p.scale2 = a.scale * 1.4426950408889634f;
    p.rows_cut = INT_MAX;
    // More tokens than sequences: some may bring enough rows for the tensor cores.
    // (When others bring none, a long one can hide behind a small count; the
    // kernel here then serves it too, in tiles of 8 or 16 rows.)
    if (v.hdp <= 128 && (long long)(a.n_tokens - a.n + 1) * p.group > kPromptRows) {
        p.rows_cut = kPromptRows;
        const cudaError_t e = tq_kv_launch_prompt(p, sms, st);
        if (e != cudaSuccess) return e;
    }
    switch (v.hdp) {
    case 64: return launch_hd<64>(p, sms, st);
    case 128: return launch_hd<128>(p, sms, st);
    default: return launch_hd<256>(p, sms, st);
    }
}
