// tq_kv_attn.cu — attention over the paged 8-bit cache (tq_kv_attention_dev;
// layout in tq_kv.h).
//
// For a query row q and the positions t that it sees, with codes k_t, v_t and
// the scales a_b, c_b of the block b that holds t:
//   s_t = (q . k_t) a_b scale log2(e),  p_t = 2^(s_t - max s_t),
//   out = sum_t p_t c_b v_t / sum_t p_t,
// in one pass over the positions with a running m, sum and accumulator.
//
// Rows. The query heads of a KV head, for all new tokens of a sequence, are the
// rows of one product, in tiles of R = 16 / PIECES rows of an m16n8k16 MMA.
// Codes are exact in float16. With PIECES = 2 a row takes two MMA rows, q = hi
// + lo (and p likewise), each a float16, which keeps 22 bits of both: float32
// products for float32 queries, at no cost while a KV head has at most 8 rows.
// With PIECES = 1 a 16-bit q is one float16 (exact: the row is scaled by a power
// of two first) and p is rounded to 11 bits: at most an eighth of a bfloat16
// output's own rounding, as much as a float16 output's (tq_kv_prompt.cu has figures).
// The value scale c_b = 2^e_b x mantissa goes with the weights, so that what a row
// gives no weight, or does not see, costs the rest no bits: m is a power of two at
// or above 2^(s_t + e_b), p_t = 2^(s_t + e_b - m), the mantissa rides on p in
// float16's range, and the sum is of p_t 2^-e_b, float32. Both powers are exact.
//
// Work. A warp takes 64 positions at a time: keys and values come by bulk copies
// of 16-position blocks into its own ring of three slots (k, v, k, ..), two of
// them in flight while one is used, and go from there straight into MMA
// fragments: sixteen dimensions of a key, or sixteen positions of a value
// dimension, are one 16-byte read, and q and p are permuted to match. The scores
// of the MMA's accumulator are the next product's operand in place.
// All (sequence, KV head, row tile) segments laid end to end, each as long as its
// tiles and, when warps have several, a unit before them for what it costs
// besides, are cut evenly over the CTAs, then over their warps, wherever the cuts fall (lengths are device data;
// every CTA makes the same sums). A warp's unfinished segments meet in its
// CTA, the CTA's in the CTA that arrives last, in a fixed order: results do not
// depend on timing.
//
// Bound. A sequence or two of ordinary length: latency, 9 us for one tile (the
// launch; lengths, page, codes one after the other from L2; a first pass through
// the code), 13 us at 2,559 positions with the joins. Many or long ones: the
// instructions between the copies. 64 sequences of 124,000 positions (28 / 4
// bfloat16 heads of 128) take 39 us, 3.3 TB/s (50% of the measured copy), 2
// sequences of 264,000 64 us, 4.2 TB/s (64%). With two warps a scheduler (248
// registers, and the rings fill shared memory; heads above 128 take all 255 and
// spill 1.2 KB) issue slots are 29% used; waiting
// for instructions is the largest stall, since a tile's straight code exceeds the
// instruction caches, then the fixed latency of one instruction after another.
#include <climits>
#include <type_traits>

#include "tq_kv_attn.cuh"

namespace {

using namespace tqkv;
using Params = TqKvParams;

constexpr int kTile = 64;       // positions per step of a warp
constexpr int kSlots = 3;       // ring slots per warp
constexpr int kWide = 4;        // MMA accumulators worked on in turn
constexpr int kMinTiles = 8;    // units per CTA below which fewer CTAs work: one for each warp
constexpr int kPromptRows = 48; // rows of a sequence above which the prompt kernel takes it
constexpr double kPromptWork = 512e6; // rows x positions x head size up to which it stays off
constexpr int kDirect = 1024;   // sequences whose lengths are kept in shared memory
constexpr int kSums = kKvSums;
constexpr float kPUnit = 16384.f; // p = 1 in float16: times a mantissa it stays below 2^15, its low piece normal
constexpr size_t kHead = kKvHead;
constexpr int kMaxGrid = kHead / sizeof(unsigned);

constexpr int warps_of(int hdp) { return hdp == 256 ? 4 : hdp == 128 ? 8 : 12; } // one CTA per SM
constexpr int slot_bytes(int hdp) { return kTile * hdp + 128; }
constexpr int value_pitch(int hdp) { return TQ_KV_BLOCK * hdp + 32; } // four blocks in distinct banks
constexpr int partial_pitch(int hdp) { return hdp + 8; } // floats of a row: two wavefronts a store
constexpr int partial_floats(int hdp) { return 16 * partial_pitch(hdp) + 32; } // sums, then m, then l
constexpr int partials_of(int hdp) { return warps_of(hdp) + 2; } // per CTA: two that others read, one for each warp
constexpr size_t smem_bytes(int hdp) {
    return (size_t)warps_of(hdp) * kSlots * slot_bytes(hdp) + sizeof(long long) * (kSums + 1) +
           sizeof(int) * (2 * kDirect + 2);
}

template <int HDP, int PIECES, typename T>
__global__ void __launch_bounds__(32 * warps_of(HDP), 1) kv_attn_kernel(const __grid_constant__ Params p) {
    constexpr int NW = warps_of(HDP), NT = 32 * NW, R = 16 / PIECES, KK = HDP / 64, NI = HDP / 8, PP = partial_pitch(HDP);
    extern __shared__ __align__(128) unsigned char sm[];
    long long *sums = reinterpret_cast<long long *>(sm + (size_t)NW * kSlots * slot_bytes(HDP));
    int *s_starts = reinterpret_cast<int *>(sums + kSums + 1), *s_lens = s_starts + kDirect + 1;
    __shared__ uint64_t bars[NW][kSlots];
    __shared__ long long s_scan[NW][2];
    __shared__ long long e_seg[2 * NW], e_end[2 * NW]; // unfinished segments of the warps: first and last tile + 1
    __shared__ int e_row[2 * NW][3];                   // their sequence, KV head, row tile
    __shared__ const float *e_at[2 * NW];              // and where their sums are
    // jobs: the first of their places in s_list, how many partials (of this CTA; wide: of all), the
    // rows before them (wide: their rows), the first CTA of a segment that others share
    struct Job {
        int at, k, row0, from;
    };
    __shared__ Job s_job[2 * NW], s_wide[2];
    __shared__ int s_list[2 * NW], s_jobs, s_rows, s_wides, s_last[2];
    __shared__ volatile int s_late[NW];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int n = p.a.n, n_kv = p.c.n_kv, group = p.group;

    // ---- lengths, checked; sums of the sequences' tiles --------------------------------
    // Up to 32 sequences: every warp makes the sums for itself, a sequence a lane.
    // Else the block makes them, the lengths and sums in shared memory.
    const bool alone = n <= 32, direct = !alone && n <= kDirect;
    if (direct) {
        for (int i = tid; i <= n; i += NT) s_starts[i] = p.a.starts[i];
        for (int i = tid; i < n; i += NT) s_lens[i] = p.a.lens[i];
    }
    if (lane < kSlots) tqp::mbar_init(&bars[warp][lane], 1);
    if (lane == 0) s_late[warp] = 0;
    if (lane < 2) e_seg[2 * warp + lane] = -1;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (alone)
        __syncwarp();
    else
        __syncthreads();
    const int *starts = direct ? s_starts : p.a.starts, *lens = direct ? s_lens : p.a.lens;
    auto seq_of = [&](int i) {
        Seq s = seq_at(p, starts, lens, i);
        if (s.nq > p.tokens_cut) s.nq = 0; // the prompt kernel's
        return s;
    };
    auto tiles_per = [](const Seq &s) { return s.len > kTile ? (s.len + kTile - 1) / kTile : 1; };
    auto row_tiles = [&](const Seq &s) { return (s.nq * group + R - 1) / R; };
    // A segment counts its tiles and, when the warps have more than one tile each,
    // another for what it costs besides. 64 sequences of 124,000 positions (28 / 4
    // heads of 128): 42 us with it, 55 without; 48 short ones: 17 with it, 14 without.
    int cost;
    auto units_of = [&](int nrt, int tps) { return (long long)nrt * n_kv * (tps + cost); };
    auto choose_cost = [&](long long tiles) { cost = tiles > (long long)gridDim.x * NW ? 1 : 0; };
    const int span = 1 << p.shift_sums, entries = (n + span - 1) >> p.shift_sums;
    long long total, lane_sum = 0; // lane_sum: units before sequence `lane`
    if (alone) {
        long long segs = 0, tiles = 0;
        if (lane < n) {
            const Seq s = seq_of(lane);
            segs = (long long)row_tiles(s) * n_kv;
            tiles = segs * tiles_per(s);
        }
        long long si = segs, ti = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, si, o), w = __shfl_up_sync(0xffffffffu, ti, o);
            if (lane >= o) si += v, ti += w;
        }
        total = __shfl_sync(0xffffffffu, ti, 31);
        choose_cost(total);
        total += cost * __shfl_sync(0xffffffffu, si, 31);
        lane_sum = ti - tiles + cost * (si - segs);
    } else { // kSums entries over NT threads
        constexpr int PER = (kSums + NT - 1) / NT;
        long long segs[PER], tiles[PER], si = 0, ti = 0;
#pragma unroll
        for (int u = 0; u < PER; u++) {
            const int e = tid * PER + u;
            segs[u] = tiles[u] = 0;
            for (int i = e << p.shift_sums; e < entries && i < min(n, (e + 1) << p.shift_sums); i++) {
                const Seq s = seq_of(i);
                const long long k = (long long)row_tiles(s) * n_kv;
                segs[u] += k;
                tiles[u] += k * tiles_per(s);
            }
            si += segs[u];
            ti += tiles[u];
        }
        const long long own_s = si, own_t = ti;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, si, o), w = __shfl_up_sync(0xffffffffu, ti, o);
            if (lane >= o) si += v, ti += w;
        }
        if (lane == 31) s_scan[warp][0] = si, s_scan[warp][1] = ti;
        __syncthreads();
        long long all_s = 0, before_s = si - own_s, before_t = ti - own_t;
        total = 0;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const long long a = s_scan[w][0], b = s_scan[w][1];
            if (w < warp) before_s += a, before_t += b;
            all_s += a, total += b;
        }
        choose_cost(total);
        total += cost * all_s;
        long long before = before_t + cost * before_s;
#pragma unroll
        for (int u = 0; u < PER; u++) {
            const int e = tid * PER + u;
            if (e <= entries) sums[e] = before;
            before += tiles[u] + cost * segs[u];
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
    // what other CTAs read lies together: few memory pages to look up
    auto partial_at = [&](int cta, int k) { return part + (size_t)(2 * cta + k) * partial_floats(HDP); };
    auto warp_partial = [&]() {
        return part + ((size_t)2 * gridDim.x + (size_t)NW * blockIdx.x + warp) * partial_floats(HDP);
    };

    struct Cursor { // a segment (sequence, KV head, row tile) and a tile of it
        int i, head, rt, nrt, tile, tps;
        int seen;      // positions that some row of it sees
        long long pos; // the tile's unit
        Seq s;
    };
    auto enter = [&](Cursor &c) { // a sequence's figures
        c.s = seq_of(c.i);
        c.tps = tiles_per(c.s);
        c.nrt = row_tiles(c.s);
    };
    auto begin = [&](Cursor &c) { // a segment's
        const int last = min((c.rt + 1) * R, c.s.nq * group) - 1;
        c.seen = min(c.s.len, max(0, c.s.len - c.s.nq + last / group + 1));
    };
    auto advance = [&](Cursor &c) { // to the next tile; its pos is at or past the list's end when there is none
        c.pos++;
        if (++c.tile < c.tps) return;
        c.tile = 0;
        c.pos += cost;
        if (++c.rt == c.nrt) {
            c.rt = 0;
            if (++c.head == n_kv) {
                c.head = 0;
                do {
                    c.i++;
                    if (c.i >= n) return;
                    enter(c);
                } while (c.nrt == 0);
            }
        }
        begin(c);
    };

    unsigned char *ring = sm + (size_t)warp * kSlots * slot_bytes(HDP);
    Cursor cur;
    if (x0 < x1) { // the first tile at or behind unit x0
        long long rest;
        if (alone) { // the last sequence that begins at or before it: the one that holds it, empty ones apart
            cur.i = 31 - __clz(__ballot_sync(0xffffffffu, lane < n && lane_sum <= x0));
            rest = x0 - __shfl_sync(0xffffffffu, lane_sum, cur.i);
        } else {
            int lo = 0, hi = entries;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (sums[mid] <= x0)
                    lo = mid;
                else
                    hi = mid;
            }
            rest = x0 - sums[lo];
            cur.i = lo << p.shift_sums;
        }
        enter(cur);
        while (rest >= units_of(cur.nrt, cur.tps)) {
            rest -= units_of(cur.nrt, cur.tps);
            cur.i++;
            enter(cur);
        }
        const int per = cur.tps + cost, seg = (int)(rest / per), in = (int)(rest - (long long)seg * per);
        cur.head = seg / cur.nrt;
        cur.rt = seg - cur.head * cur.nrt;
        cur.tile = max(0, in - cost);
        cur.pos = x0 + max(0, cost - in);
        begin(cur);
    }
    if (x0 < x1 && cur.pos < x1) {
        // ---- the loader: one tile's keys, then its values; item = 2 * tile number + (0 | 1) --
        Cursor ld = cur;
        unsigned item = 0;
        struct Next { // this lane's block (t) of a tile: its page (< 0: not there), KV head, place in the page
            int id, head, in;
            bool some; // whether there is such a tile
        };
        auto ask = [&]() { // the next tile's; its page is on its way
            Next b{-1, 0, 0, ld.pos < x1};
            if (!b.some) return b;
            const int pos = ld.tile * kTile + t * TQ_KV_BLOCK;
            b.head = ld.head;
            b.in = (pos & (p.c.page - 1)) >> 4;
            if (pos < ld.seen) {
                b.id = p.a.table[(size_t)ld.i * p.a.table_stride + (pos >> p.c.page_shift)];
                if ((unsigned)b.id >= (unsigned)p.c.n_pages) b.id = -2;
            }
            advance(ld);
            return b;
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
        Next n0 = ask(), n1 = ask(), nv = n0; // the next tiles for keys, the next for values
        auto load_keys = [&](float2 &sc) { // and this lane's block's scales; x < 0: a block that is not there
            sc = make_float2(-1.f, 0.f);
            if (!n0.some) return;
            if (n0.id == -2) atomicOr(p.c.status, TQ_KV_STATUS_PAGE);
            copy(p.c.k, n0.id, n0.head, n0.in, TQ_KV_BLOCK * HDP);
            if (n0.id >= 0) sc = __ldg(p.c.scale + (size_t)n0.id * n_kv + n0.head);
            nv = n0, n0 = n1, n1 = ask();
        };
        auto load_values = [&]() { copy(p.c.v, nv.id, nv.head, nv.in, value_pitch(HDP)); };

        float2 sc, sc_next;
        unsigned used = 0; // items used

        unsigned qf[KK][4][4];
        float O[NI][4];
        float m[2], l[2], row_unit[2];
        int lim[2], least = 0;
        long long seg_from = 0;
        auto start = [&](const Cursor &now) { // a segment: its queries, and nothing seen yet
            seg_from = now.pos - now.tile;
            least = min(now.s.len, max(0, now.s.len - now.s.nq + now.rt * R / group + 1));
#pragma unroll
            for (int h = 0; h < 2; h++) {
                m[h] = -INFINITY;
                l[h] = 0.f;
                row_unit[h] = 1.f;
                lim[h] = now.s.len;
            }
#pragma unroll
            for (int i = 0; i < NI; i++) O[i][0] = O[i][1] = O[i][2] = O[i][3] = 0.f;
#pragma unroll
            for (int h = 0; h < 3 - PIECES; h++) { // MMA rows g and, with one piece, g + 8
                const int row = now.rt * R + g + 8 * h;
                const int tok = row / group, hq = now.head * group + row - tok * group;
                const bool live = row < now.s.nq * group;
                const T *q = static_cast<const T *>(p.a.q) + (size_t)(now.s.start + tok) * p.a.q_stride +
                             (size_t)hq * p.c.hd + 16 * t;
                constexpr int E = 16 / sizeof(T), W = 16 / E; // words of the lane's sixteen dimensions
                uint4 x[KK][W];
                if (p.vec) {
#pragma unroll
                    for (int kk = 0; kk < KK; kk++)
#pragma unroll
                        for (int j = 0; j < W; j++)
                            x[kk][j] = live && 64 * kk + 16 * t + E * j < p.c.hd
                                           ? __ldg(reinterpret_cast<const uint4 *>(q + 64 * kk + E * j))
                                           : make_uint4(0, 0, 0, 0);
                } else {
#pragma unroll
                    for (int kk = 0; kk < KK; kk++)
#pragma unroll
                        for (int j = 0; j < W; j++)
#pragma unroll
                            for (int u = 0; u < E; u++)
                                reinterpret_cast<T *>(&x[kk][j])[u] =
                                    live && 64 * kk + 16 * t + E * j < p.c.hd ? q[64 * kk + E * j + u] : T(0.f);
                }
                float big = 0.f;
#pragma unroll
                for (int kk = 0; kk < KK; kk++)
#pragma unroll
                    for (int u = 0; u < 16; u++)
                        big = fmaxf(big, fabsf(Elem<T>::get(reinterpret_cast<const T *>(&x[kk][0]) + u)));
                big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
                big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
                float unit = row_scale(big, &row_unit[h]);
                if (p.scale2 < 0.f) unit = -unit; // the block factors stay positive
                if (live) lim[h] = min(now.s.len, max(0, now.s.len - now.s.nq + tok + 1));
#pragma unroll
                for (int kk = 0; kk < KK; kk++)
#pragma unroll
                    for (int u = 0; u < 4; u++)
#pragma unroll
                        for (int e = 0; e < 2; e++) { // dimensions 4u + 2e, + 1 of the lane's sixteen
                            const T *y = reinterpret_cast<const T *>(&x[kk][0]) + 4 * u + 2 * e;
                            const float y0 = Elem<T>::get(y) * unit, y1 = Elem<T>::get(y + 1) * unit;
                            const unsigned hi = pack2(y0, y1);
                            qf[kk][u][2 * e + h] = hi;
                            if (PIECES == 2) {
                                const float2 b = unpack2(hi);
                                qf[kk][u][2 * e + 1] = pack2(y0 - b.x, y1 - b.y);
                            }
                        }
            }
            if (PIECES == 2) lim[1] = lim[0];
        };
        start(cur);
        load_keys(sc);
        load_values();
        load_keys(sc_next);
        for (bool more = true, fresh = false; more;) {
            const int head = cur.head, rt = cur.rt;
            const Cursor now = cur;
            advance(cur);
            more = cur.pos < x1;
            if (fresh) start(now);
            fresh = false;
            // ---- s = q . k for 64 positions ----
            const int pos0 = now.tile * kTile;
            float S[8][4];
#pragma unroll
            for (int j = 0; j < 8; j++) S[j][0] = S[j][1] = S[j][2] = S[j][3] = 0.f;
            wait_slot(&bars[warp][used % kSlots], (used / kSlots) & 1, &s_late[warp], p.c.status);
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
            if (more) load_values();
            // ---- softmax of the lane's 16 positions (its block), per row ----
            const bool there = sc.x >= 0.f || sc.x != sc.x;
            const bool whole = pos0 + kTile <= least && __all_sync(0xffffffffu, there);
            const float a = there ? sc.x * fabsf(p.scale2) : 0.f, c = there ? sc.y : 0.f;
            // c = 2^lift x its mantissa, which rides on p in units of kPUnit; drop = 2^-lift
            const bool valued = c >= kLeastValue;
            const unsigned power = __float_as_uint(valued ? c : kNoValue) & 0x7f800000u;
            const float lift = (float)((int)(power >> 23) - 127);
            const float drop = __uint_as_float(max(0x7f000000u - power, 0x00400000u)); // 2^-127 has no exponent
            const float ride = valued ? kPUnit * __uint_as_float((__float_as_uint(c) & 0x007fffffu) | 0x3f800000u)
                                      : c != c ? c : 0.f;
            constexpr int H = 3 - PIECES;
            float alpha[2];
            unsigned pf[4][4];
#pragma unroll
            for (int h = 0; h < H; h++) {
                // a block that the row sees nothing of has the factors of one that is not there: 0 times a NaN is no 0
                const bool none = !there || pos0 + 16 * t >= lim[h];
                const float af = none ? 0.f : a * row_unit[h], low = af < kLeast ? kLeast : af; // a NaN stays
                const float r = none ? 0.f : ride;
                float f = low, v[16], mx = -INFINITY;
#pragma unroll
                for (int j = 0; j < 8; j++)
#pragma unroll
                    for (int e = 0; e < 2; e++) v[2 * j + e] = PIECES == 2 ? S[j][e] + S[j][2 + e] : S[j][2 * h + e];
                if (!whole) {
#pragma unroll
                    for (int j = 0; j < 16; j++)
                        if (!there || pos0 + 16 * t + j >= lim[h]) v[j] = -INFINITY;
                }
#pragma unroll
                for (int j = 0; j < 16; j++) mx = fmaxf(mx, v[j]);
                mx = fmaf(mx, f, lift);
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float m1 = fmaxf(m[h], ceilf(mx)), base = m1 == -INFINITY ? 0.f : m1;
                float off = lift - base;
                alpha[h] = ex2(m[h] - base);
                m[h] = m1;
                if (fabsf(base) >= kFar) { // m was rounded: so is what it is compared with
#pragma unroll
                    for (int j = 0; j < 16; j++) v[j] = __fadd_rn(fmaf(v[j], f, lift), -base);
                    f = 1.f, off = 0.f;
                }
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    v[j] = ex2(fmaf(v[j], f, off));
                    sum += v[j];
                    v[j] *= r;
                }
                l[h] = fmaf(sum, drop, l[h] * alpha[h]);
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
            wait_slot(&bars[warp][used % kSlots], (used / kSlots) & 1, &s_late[warp], p.c.status);
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
            const bool ends = now.tile + 1 == now.tps;
            if (ends || !more) {
                constexpr float unit = 1.f / kPUnit;
#pragma unroll
                for (int h = 0; h < H; h++) {
                    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
                    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
                }
                const bool began = seg_from >= x0;
                const int rows = now.s.nq * group;
                if (ends && began) {
#pragma unroll
                    for (int h = 0; h < H; h++) {
                        const int row = rt * R + g + 8 * h;
                        if (row >= rows) continue;
                        const int tok = row / group, hq = head * group + row - tok * group;
                        T *o = static_cast<T *>(p.a.out) + (size_t)(now.s.start + tok) * p.a.out_stride +
                               (size_t)hq * p.c.hd;
                        const float inv = l[h] == 0.f ? 0.f : unit / l[h];
#pragma unroll
                        for (int i = 0; i < NI; i++) {
                            const int d = 8 * i + 2 * t;
                            const float y0 = PIECES == 2 ? O[i][0] + O[i][2] : O[i][2 * h];
                            const float y1 = PIECES == 2 ? O[i][1] + O[i][3] : O[i][2 * h + 1];
                            if (d < p.c.hd) Elem<T>::put2(o + d, y0 * inv, y1 * inv, p.vec);
                        }
                    }
                } else { // to be joined: sums in plain units, m and l
                    // the warp's last: over its ring, which is through; else the workspace
                    const int e = 2 * warp + (began ? 1 : 0);
                    float *to = !more ? reinterpret_cast<float *>(ring) : warp_partial();
#pragma unroll
                    for (int h = 0; h < H; h++) {
#pragma unroll
                        for (int i = 0; i < NI; i++) {
                            const float y0 = PIECES == 2 ? O[i][0] + O[i][2] : O[i][2 * h];
                            const float y1 = PIECES == 2 ? O[i][1] + O[i][3] : O[i][2 * h + 1];
                            *reinterpret_cast<float2 *>(to + (g + 8 * h) * PP + 8 * i + 2 * t) =
                                make_float2(y0 * unit, y1 * unit);
                        }
                        if (t == 0) {
                            to[16 * PP + g + 8 * h] = m[h];
                            to[16 * PP + 16 + g + 8 * h] = l[h];
                        }
                    }
                    if (lane == 0) {
                        e_seg[e] = seg_from;
                        e_end[e] = seg_from + now.tps;
                        e_row[e][0] = now.i;
                        e_row[e][1] = head;
                        e_row[e][2] = rt;
                        e_at[e] = to;
                    }
                }
                fresh = true;
            }
        }
    }
    __syncthreads();

    // ---- join the warps' unfinished segments, then the CTAs' ------------------------------
    // The places in use, in order: a segment's are neighbours, and make a job. Its
    // rows are joined a warp each, so that many short segments go side by side.
    if (warp == 0) {
        const bool used = lane < 2 * NW && e_seg[lane] >= 0;
        const unsigned all = __ballot_sync(0xffffffffu, used), below = (1u << lane) - 1;
        if (used) s_list[__popc(all & below)] = lane;
        __syncwarp();
        const int count = __popc(all), e = lane < count ? s_list[lane] : 0;
        const long long seg = lane < count ? e_seg[e] : -1, before = __shfl_up_sync(0xffffffffu, seg, 1);
        const bool first = lane < count && (lane == 0 || seg != before);
        const unsigned firsts = __ballot_sync(0xffffffffu, first);
        int rows = 0;
        if (first) rows = min(R, seq_of(e_row[e][0]).nq * group - e_row[e][2] * R);
        int upto = rows;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const bool wide = first && (seg < c0 || e_end[e] > c1); // other CTAs share it: this CTA's first or last
        const unsigned wides = __ballot_sync(0xffffffffu, wide);
        if (first) {
            Job &b = s_job[__popc(firsts & below)];
            b.at = lane;
            b.k = (firsts & ~below & ~(1u << lane) ? __ffs(firsts & ~below & ~(1u << lane)) - 1 : count) - lane;
            b.row0 = upto - rows;
            b.from = wide ? split.owner(seg) : -1;
            if (wide) {
                Job &w = s_wide[__popc(wides & below)];
                w.at = lane;
                w.from = b.from;
                w.k = split.owner(e_end[e] - 1) - b.from + 1;
                w.row0 = rows;
            }
        }
        if (lane == 31) s_rows = upto;
        if (lane == 0) s_jobs = __popc(firsts), s_wides = __popc(wides);
    }
    __syncthreads();
    if (s_jobs == 0) return;
    // The sum of row r over k partials, partial(j), by a warp: to a partial or, without one, to the output.
    // mine: partials of this CTA, in shared memory or the workspace.
    auto join_row = [&](auto partial, auto mine, int k, int r, int e, float *to) {
        constexpr int kAhead = 8; // partials on their way at once
        const int i = e_row[e][0], head = e_row[e][1], row = e_row[e][2] * R + r;
        const int tok = row / group, hq = head * group + row - tok * group;
        T *o = static_cast<T *>(p.a.out) + (size_t)(seq_of(i).start + tok) * p.a.out_stride + (size_t)hq * p.c.hd;
        for (int d = 4 * lane; d < HDP; d += 128) {
            float M = -INFINITY, L = 0.f;
            float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
            for (int j0 = 0; j0 < k; j0 += kAhead) {
                float m[kAhead], l[kAhead], top = M;
                float4 y[kAhead];
#pragma unroll
                for (int u = 0; u < kAhead; u++) { // the last again, at no weight, beyond the end
                    const float *f = partial(min(j0 + u, k - 1));
                    if constexpr (mine.value) {
                        m[u] = f[16 * PP + r];
                        l[u] = f[16 * PP + 16 + r];
                        y[u] = *reinterpret_cast<const float4 *>(f + r * PP + d);
                    } else {
                        m[u] = __ldcg(f + 16 * PP + r);
                        l[u] = __ldcg(f + 16 * PP + 16 + r);
                        y[u] = __ldcg(reinterpret_cast<const float4 *>(f + r * PP + d));
                    }
                    if (j0 + u >= k) m[u] = -INFINITY;
                }
#pragma unroll
                for (int u = 0; u < kAhead; u++) top = fmaxf(top, m[u]);
                const float base = top == -INFINITY ? 0.f : top, old = exp2f(M - base);
                M = top;
                L *= old, A.x *= old, A.y *= old, A.z *= old, A.w *= old;
#pragma unroll
                for (int u = 0; u < kAhead; u++) {
                    const float w = exp2f(m[u] - base);
                    L += w * l[u];
                    A.x += w * y[u].x;
                    A.y += w * y[u].y;
                    A.z += w * y[u].z;
                    A.w += w * y[u].w;
                }
            }
            if (to) {
                *reinterpret_cast<float4 *>(to + r * PP + d) = A;
                if (d == 0) to[16 * PP + r] = M, to[16 * PP + 16 + r] = L;
            } else if (d < p.c.hd) {
                const float inv = L == 0.f ? 0.f : 1.f / L;
                Elem<T>::put2(o + d, A.x * inv, A.y * inv, p.vec);
                Elem<T>::put2(o + d + 2, A.z * inv, A.w * inv, p.vec);
            }
        }
    };
    for (int item = warp; item < s_rows; item += NW) {
        const Job b = s_job[__popc(__ballot_sync(0xffffffffu, lane < s_jobs && s_job[lane < s_jobs ? lane : 0].row0 <= item)) - 1];
        float *to = b.from < 0 ? nullptr : partial_at(blockIdx.x, (int)blockIdx.x == b.from ? 1 : 0);
        join_row([&](int j) { return e_at[s_list[b.at + j]]; }, std::true_type(), b.k, item - b.row0, s_list[b.at], to);
    }
    if (s_wides == 0) return;
    __syncthreads(); // the partials are written
    unsigned *counters = static_cast<unsigned *>(p.a.workspace);
    if (tid < s_wides) s_last[tid] = tq_arrive_last(counters + s_wide[tid].from, s_wide[tid].k);
    __syncthreads();
    const int rows0 = s_last[0] ? s_wide[0].row0 : 0, rows1 = s_wides > 1 && s_last[1] ? s_wide[1].row0 : 0;
    for (int item = warp; item < rows0 + rows1; item += NW) {
        const Job b = s_wide[item < rows0 ? 0 : 1];
        join_row([&](int j) { return (const float *)partial_at(b.from + j, j == 0 ? 1 : 0); }, std::false_type(), b.k,
                 item < rows0 ? item : item - rows0, s_list[b.at], nullptr);
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
    const int grid = min(kMaxGrid, sms);
    kv_attn_kernel<HDP, PIECES, T><<<grid, 32 * warps_of(HDP), smem_bytes(HDP), st>>>(p);
    return cudaGetLastError();
}

template <int HDP> cudaError_t launch_hd(const Params &p, int sms, cudaStream_t st) {
    // Two pieces keep float32's precision; a 16-bit query takes one piece when its
    // rows of one token would not fit the eight that two pieces leave. One piece
    // everywhere: 16 sequences of 4096, 28 / 4 bfloat16 heads, 2 tokens 35 us in
    // place of 41, but one of 512 positions 21 in place of 16 and less exact.
    const bool two = p.a.dtype == TQ_LINEAR_F32 || p.group <= 8;
    if (p.a.dtype == TQ_LINEAR_F32) return launch<HDP, 2, float>(p, sms, st);
    if (p.a.dtype == TQ_LINEAR_F16) return two ? launch<HDP, 2, __half>(p, sms, st) : launch<HDP, 1, __half>(p, sms, st);
    return two ? launch<HDP, 2, __nv_bfloat16>(p, sms, st) : launch<HDP, 1, __nv_bfloat16>(p, sms, st);
}

} // namespace

static size_t small_workspace(int hdp, int sms) {
    const size_t grid = (size_t)(sms < kMaxGrid ? sms : kMaxGrid);
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
    p.tokens_cut = INT_MAX;
    // More tokens than sequences: some may bring enough rows for the tensor cores.
    // (When others bring none, a long one can hide behind a small count; the
    // kernel here then serves it too, in tiles of 8 or 16 rows.)
    // Both sides, 28 query heads of 128 on 4 KV heads, bfloat16, in microseconds
    // here / there:
    //   16 sequences of 4096: 28 rows 65 / 73, 42 rows 89 / 72, 98 rows 175 / 77;
    //   16 sequences of 512 (1.4e6 to 9e6 rows x positions): 28 rows 21 / 37,
    //   98 rows 42 / 39, 126 rows 47 / 40, 259 rows 74 / 67;
    //   one of 4096 (at most 15e6): 196 rows 35 / 62, 448 rows 59 / 65, 896 rows 101 / 66.
    // So the rows decide between them, and the other kernel's fixed time (its
    // set-up, its second kernel and, for a whole call, this one after it) is worth
    // it from about 4e6 rows x positions on at a head size of 128. The host knows no
    // lengths: the table's width stands for them.
    const double work = (double)a.n_tokens * a.n_q * a.table_cols * v.page * v.hdp;
    if (v.hdp <= 128 && (long long)(a.n_tokens - a.n + 1) * p.group > kPromptRows && work > kPromptWork) {
        p.tokens_cut = kPromptRows / p.group;
        const cudaError_t e = tq_kv_launch_prompt(p, sms, st);
        if (e != cudaSuccess) return e;
    }
    switch (v.hdp) {
    case 64: return launch_hd<64>(p, sms, st);
    case 128: return launch_hd<128>(p, sms, st);
    default: return launch_hd<256>(p, sms, st);
    }
}
