// The split pass of attn_shared.cu as a device function: it runs in a launch of its own, or on CTAs of the prefix kernel's launch
// (attn_shared_prefix.cu). Mathematics, tiles and figures are described there.
#pragma once

#include <cuda.h>

#include <cmath>
#include <type_traits>

#include "attn_internal.cuh"
#include "ptx_sm100.cuh"
#include "tcgen05_sm100.cuh"
#include "tma_tile.cuh"

namespace b200 {

constexpr int kSplitConsumers = 128;  // threads that multiply
constexpr int kTilePairs = 64;  // (row, head) pairs of a tile
constexpr uint32_t kMaxBatch = 2048;
constexpr uint32_t kMaxSlots = 12;
constexpr size_t kSplitSmem = 113 * 1024;  // of a CTA of the split pass, two per SM

// How the four warps share a tile of one kind of segment: hpc heads x wm blocks of 16 query rows x ts shares of the keys = 4.
struct Shape {
    uint32_t hpc, wm, ts;
    uint32_t keys;    // of a tile: 64 / hpc
    uint32_t groups;  // n_kv_heads / hpc
    uint32_t rec_rows;  // query rows per (piece, share of keys, head): 16 * wm for the prefix, G for own rows
};

struct SharedParams {
    const uint16_t* q;
    const uint32_t* kv_len;
    uint32_t kv_len_uniform;
    uint32_t batch, n_heads, n_kv_heads, group;
    uint32_t div_heads, div_group;  // divider(n_heads), divider(group)
    uint32_t prefix, rows;
    float scale_log2;       // of the scale's magnitude
    uint32_t q_sign;        // 0x80008000 for a negative scale: flips the query's sign instead
    Shape pre, own;
    uint32_t row_blocks;    // blocks of 16 * pre.wm query rows against the prefix
    uint32_t prefix_segs;   // pre.groups * row_blocks; 0 in the split pass when another kernel takes the prefix
    uint32_t prefix_tiles;  // of one such segment
    float* part_pre;        // [(grid + prefix_segs) * ts * hpc][rec_rows][D]
    float* lse_pre;
    float* part_own;        // [(grid + batch * groups) * ts * hpc][rec_rows][D]
    float* lse_own;
    uint32_t* seg_pre;      // [prefix_segs] segment_ctas() words
    uint32_t* seg_own;      // [batch * own.groups]
    float* raw;             // [batch][n_heads][raw_stride] scaled scores in log2 units, or null
    uint64_t raw_stride;
    uint32_t* status;
    uint32_t prefix_weight; // cost of a prefix tile in own tiles
    uint32_t switch_units;  // cost of an own segment's start in own tiles
    uint32_t slots, q_held; // ring slots (K or V of a tile each), query rows a warp keeps in shared memory
    uint32_t ctas;          // CTAs of the split pass
    // merge
    void* o;
    float* lse;
    int32_t o_dtype;
    const float* scores;
    float* scores_out;
    uint64_t score_stride, score_out_stride;
    uint32_t out_ctas, score_chunks, score_rows;  // score_rows: of a CTA that adds up weights
};

__device__ __forceinline__ uint32_t own_len(const SharedParams& p, uint32_t b) {
    return min(p.kv_len ? p.kv_len[b] : p.kv_len_uniform, p.rows);
}

// A tile of the list and its segment.
struct Cursor {
    uint32_t own, seg;         // kind; index among the segments of its kind
    uint32_t b, hg, rb;        // own: sequence; head group; prefix: block of query rows
    uint32_t tile, tiles, len;
    uint32_t unit;             // the tile's first unit of the list
};

constexpr int kSplitThreads = kSplitConsumers + 64;  // four consumer warps, the producer warp, one that notes which CTAs share each segment

// CTA `cta` of p.ctas, kSplitThreads threads of a block numbered from 0 by tid, with the shared memory at smem_raw and the barriers
// bar0 and bar0 + 1 of the block to themselves.
template <int D, bool BF16, bool RES>
__device__ __forceinline__ void split_body(const CUtensorMap& tm_k, const CUtensorMap& tm_v, const CUtensorMap& tm_kp, const CUtensorMap& tm_vp,
                                           const SharedParams& p, unsigned char* smem_raw, const uint32_t cta, const int tid, const int bar0) {
    constexpr int kParts = D / 64;                    // 128-byte parts of a head's row
    constexpr uint32_t kPartBytes = kTilePairs * 128;    // of all heads and keys of a tile
    constexpr uint32_t kSlotBytes = kParts * kPartBytes; // K or V of a tile
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);  // swizzled tiles want 1024-byte alignment
    const uint32_t ring = smem_u32(smem);
    const uint32_t slots = p.slots;
    const uint32_t bars = ring + slots * kSlotBytes;          // full [slots], empty [slots]
    const uint32_t q_zero = bars + kMaxSlots * 16;            // a row of zeros
    const uint32_t q_rows = q_zero + D * 2;                   // [4 warps][q_held rows], 16-byte chunks swizzled by the row
    uint32_t* s_cum = reinterpret_cast<uint32_t*>(smem + (q_rows - ring) + 4 * p.q_held * D * 2);  // [batch + 1] units of own rows, one head group
    uint32_t* s_warp = s_cum + p.batch + 1;                   // [6]
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    if (tid == 0) {
        for (uint32_t i = 0; i < slots; ++i) {
            mbar_init(bars + 8 * i, 1);
            mbar_init(bars + 8 * (slots + i), 4);
        }
        mbar_init_fence();
        prefetch_tensor_map(&tm_k);
        prefetch_tensor_map(&tm_v);
        if (p.prefix_segs) {
            prefetch_tensor_map(&tm_kp);
            prefetch_tensor_map(&tm_vp);
        }
    }
    if (tid < kParts * 8) st_shared_zero16(q_zero + tid * 16);
    grid_dep_launch_dependents();
    grid_dep_wait();

    // ---- units of each sequence and head group, summed up: as many sequences as threads at a time
    auto own_units = [&](uint32_t b) {
        const uint32_t tiles = (own_len(p, b) + p.own.keys - 1) / p.own.keys;
        return tiles ? tiles + p.switch_units : 0u;
    };
    {
        uint32_t base = 0;
        if (tid == 0) s_cum[0] = 0;
        for (uint32_t b0 = 0; b0 < p.batch; b0 += kSplitThreads) {
            const uint32_t b = b0 + tid;
            const uint32_t n = b < p.batch ? own_units(b) : 0u;
            if (b < p.batch && p.kv_len && p.kv_len[b] > p.rows && p.status && cta == 0) atomicOr(p.status, ATTN_STATUS_BAD_SHAPE);
            uint32_t incl = n;
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const uint32_t o = __shfl_up_sync(0xffffffffu, incl, d);
                if (lane >= d) incl += o;
            }
            if (lane == 31) s_warp[warp] = incl;
            block_wait(bar0, kSplitThreads);
            uint32_t before = base;
            for (int w = 0; w < warp; ++w) before += s_warp[w];
            if (b < p.batch) s_cum[b + 1] = before + incl;
            base += s_warp[0] + s_warp[1] + s_warp[2] + s_warp[3] + s_warp[4] + s_warp[5];
            block_wait(bar0, kSplitThreads);
        }
    }
    // The list in units: a prefix tile counts as many as its blocks of 16 query rows make it cost, an own tile one, the start of an own
    // segment (its query rows, its piece) switch_units. A tile belongs to the CTA that has its first unit; with at least a prefix tile's
    // units per CTA, every CTA between those of a segment's first and last tile has a tile of it.
    const uint32_t pre_units = p.prefix_segs * p.prefix_tiles * p.prefix_weight;
    const uint32_t units = pre_units + s_cum[p.batch] * p.own.groups;
    const uint32_t active = active_ctas(p.ctas, 0, p.prefix_segs ? p.prefix_weight : 1, units);
    uint32_t u0 = 0, u1 = 0;
    if (cta < active) {
        u0 = static_cast<uint32_t>(div_mostly_32(static_cast<uint64_t>(cta) * units, active));
        u1 = static_cast<uint32_t>(div_mostly_32((cta + 1ull) * units, active));
    }

    // The first tile at or behind unit u: its segment, and c.unit, the tile's first unit (which may be behind the CTA's last).
    auto locate = [&](uint32_t u, Cursor& c) {
        if (u < pre_units) {
            const uint32_t tile = (u + p.prefix_weight - 1) / p.prefix_weight;
            c.unit = tile * p.prefix_weight;
            if (c.unit < pre_units) {
                c.own = 0;
                c.seg = tile / p.prefix_tiles;
                c.tile = tile - c.seg * p.prefix_tiles;
                c.tiles = p.prefix_tiles;
                c.hg = c.seg / p.row_blocks;
                c.rb = c.seg - c.hg * p.row_blocks;
                c.b = 0;
                c.len = p.prefix;
                return;
            }
            u = pre_units;
        }
        c.unit = units;
        if (u >= units) return;
        const uint32_t f = u - pre_units;
        uint32_t lo = 0, hi = p.batch;  // the last sequence whose units start at or before f
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (s_cum[mid] * p.own.groups <= f) lo = mid;
            else hi = mid;
        }
        const uint32_t span = s_cum[lo + 1] - s_cum[lo];  // units of one head group
        const uint32_t r = f - s_cum[lo] * p.own.groups;
        c.own = 1;
        c.b = lo;
        c.tiles = span - p.switch_units;
        c.hg = r / span;
        const uint32_t at = max(r - c.hg * span, p.switch_units);
        c.tile = at - p.switch_units;
        c.unit = pre_units + s_cum[lo] * p.own.groups + c.hg * span + at;
        c.seg = lo * p.own.groups + c.hg;
        c.rb = 0;
        c.len = own_len(p, lo);
    };
    // the next tile of the list
    auto advance = [&](Cursor& c) {
        const uint32_t next = c.unit + (c.own ? 1 : p.prefix_weight);
        if (++c.tile < c.tiles) c.unit = next;
        else locate(next, c);
    };
    Cursor cur;  // of the consumers, and of the producer
    locate(u0, cur);
    const bool busy = cur.unit < u1;

    if (warp == 4) {
        // =============================== producer ===============================
        // 28 MB of tiles are requested at once as soon as the CTAs know theirs, and query rows that are requested behind them came 3 to
        // 5 us later, with no tile worked on until then: the consumers' requests go first.
        if (busy) block_wait(bar0 + 1, kSplitConsumers + 32);
        if (lane == 0 && busy) {
            const uint64_t once = l2_policy_evict_first();  // own rows are read once; the prefix's may be read by several blocks of rows
            const uint64_t again = l2_policy_evict_last();
            Cursor& c = cur;
            uint32_t st = 0, phase = 1;  // (a fresh barrier counts as past its odd phase: the first round does not wait)
            bool ok = true;
            while (c.unit < u1 && ok) {
                const Shape& sh = c.own ? p.own : p.pre;
                const int row = static_cast<int>(c.tile * sh.keys), head = static_cast<int>(c.hg * sh.hpc), seq = static_cast<int>(c.b);
                const uint64_t policy = c.own || p.row_blocks == 1 ? once : again;
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    if (!mbar_wait(bars + 8 * (slots + st), phase)) { ok = false; break; }
                    mbar_arrive_expect_tx(bars + 8 * st, kSlotBytes);
                    tma_load_5d_hint(ring + st * kSlotBytes, c.own ? (v ? &tm_v : &tm_k) : (v ? &tm_vp : &tm_kp), bars + 8 * st, row, head, 0, seq, policy);
                    if (++st == slots) st = 0, phase ^= 1;
                }
                advance(c);
            }
            if (!ok) {  // report, and leave no copy in flight into this CTA's memory
                if (p.status) atomicOr(p.status, ATTN_STATUS_WAIT_TIMEOUT);
                for (uint32_t i = 0; i < slots; ++i) {
                    (void)mbar_wait(bars + 8 * st, phase);
                    if (++st == slots) st = 0, phase ^= 1;
                }
            }
        }
        __syncwarp();
    } else if (warp == 5) {
        // which CTAs share each segment, for the merge pass
        const uint32_t own_segs = p.batch * p.own.groups;
        for (uint32_t s = cta * 32 + lane; s < p.prefix_segs + own_segs; s += p.ctas * 32) {
            uint32_t first, last;  // units of the first and the last tile; no tile: last < first
            if (s < p.prefix_segs) {
                first = s * p.prefix_tiles * p.prefix_weight;
                last = first + (p.prefix_tiles - 1) * p.prefix_weight;
            } else {
                const uint32_t b = (s - p.prefix_segs) / p.own.groups, hg = (s - p.prefix_segs) - b * p.own.groups;
                const uint32_t span = s_cum[b + 1] - s_cum[b], start = pre_units + s_cum[b] * p.own.groups + hg * span;
                first = span ? start + p.switch_units : 1;
                last = span ? start + span - 1 : 0;
            }
            const uint32_t from = last < first ? 0 : cta_of_tile(first, units, active);
            const uint32_t count = last < first ? 0 : cta_of_tile(last, units, active) - from + 1;
            (s < p.prefix_segs ? p.seg_pre[s] : p.seg_own[s - p.prefix_segs]) = from | count << 16;
        }
    } else {
        // =============================== consumers ===============================
        const uint32_t my_q = q_rows + warp * p.q_held * (D * 2);
        // Offsets of the 16-byte chunks that this lane hands to ldmatrix, four of them in a 128-byte part: keys, values, query row.
        uint32_t k_off[4], v_off[4], q_off[4], q_lane = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            k_off[i] = ((i * 2 + ((lane >> 3) & 1)) ^ (lane & 7)) << 4;
            v_off[i] = ((i * 2 + (lane >> 4)) ^ (lane & 7)) << 4;
            q_off[i] = 0;
        }
        float o[D / 8][4];
        float m[2], l[2];
        bool fresh = true;  // the next tile begins a run of a segment
        uint32_t slot = 0, phase = 0;
        auto next_slot = [&]() {
            if (++slot == slots) slot = 0, phase ^= 1;
        };
        bool ok = true, first_run = true;
        while (cur.unit < u1) {
            const Shape& sh = cur.own ? p.own : p.pre;
            // this warp's place: head hs of the group, block wr of query rows, share wk of the keys (all powers of two)
            const uint32_t hs = warp & (sh.hpc - 1), wr = (warp >> (sh.hpc >> 1)) & (sh.wm - 1), wk = warp >> ((sh.hpc >> 1) + (sh.wm >> 1));
            const uint32_t kvh = cur.hg * sh.hpc + hs;
            if (fresh) {
                // ---- the warp's query rows into shared memory (its own: no other warp waits); rows that are not there are the row of zeros
                fresh = false;
                const uint32_t row0 = cur.own ? wr * 16 : cur.rb * sh.wm * 16 + wr * 16, all = cur.own ? p.group : p.batch * p.group;
                const uint32_t n = row0 < all ? min(16u, all - row0) : 0u;
                auto q_at = [&](uint32_t r, uint32_t ch) {  // chunk ch of the warp's row r
                    const uint32_t row = row0 + r, b = cur.own ? cur.b : fast_div(row, p.div_group), g = cur.own ? row : row - b * p.group;
                    return p.q + (static_cast<size_t>(b) * p.n_heads + kvh * p.group + g) * D + ch * 8;
                };
                __syncwarp();
                for (uint32_t i = lane; i < n * (kParts * 8); i += 32) {
                    const uint32_t r = i / (kParts * 8), ch = i % (kParts * 8);
                    cp_async16(my_q + r * (D * 2) + ((ch ^ (r & 7)) << 4), q_at(r, ch));
                }
                if (first_run) {
                    first_run = false;
                    block_arrive(bar0 + 1, kSplitConsumers + 32);
                }
                cp_async_wait_all();
                if (p.q_sign)  // a negative scale's sign; each lane its own chunks
                    for (uint32_t i = lane; i < n * (kParts * 8); i += 32)
                        xor_shared16(my_q + i / (kParts * 8) * (D * 2) + (((i % (kParts * 8)) ^ (i / (kParts * 8) & 7)) << 4), p.q_sign);
                __syncwarp();
                const uint32_t r = lane & 15;
                q_lane = r < n ? my_q + r * (D * 2) : q_zero;
                // the next segment's rows, requested into L2, from where cp.async takes them (rows of the list's own segments follow one another in q)
                if (cur.own && cur.unit + (cur.tiles - cur.tile) < u1) {
                    const uint64_t next = static_cast<uint64_t>(cur.b) * p.n_heads + (kvh + sh.hpc) * p.group + row0;
                    for (uint32_t i = lane; i < n * kParts * 4; i += 32)  // 32 bytes each
                        if (next + i / (kParts * 4) < static_cast<uint64_t>(p.batch) * p.n_heads) touch(p.q + next * D + i * 16);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) q_off[i] = ((i * 2 + (lane >> 4)) ^ (r < n ? r & 7 : 0)) << 4;
#pragma unroll
                for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
                m[0] = m[1] = -INFINITY;
                l[0] = l[1] = 0.f;
            }
            const uint32_t head_base = hs * (sh.keys * 128);
            const uint32_t steps = sh.wm;  // 16 keys each: 64 / hpc / ts = 16 wm
            const uint32_t first0 = cur.tile * sh.keys + wk * steps * 16;  // the warp's first key in the cache
            const uint32_t live = first0 < cur.len ? min(steps, (cur.len - first0 + 15) / 16) : 0u;
            const uint32_t k_slot = slot, k_phase = phase;
            next_slot();
            const uint32_t v_slot = slot, v_phase = phase;
            next_slot();
            const uint32_t kbase = ring + k_slot * kSlotBytes + head_base, vbase = ring + v_slot * kSlotBytes + head_base;
            ok = mbar_wait(bars + 8 * k_slot, k_phase);
            // Scores, probabilities and products of NB blocks of 16 keys.
            auto blocks = [&](auto nb, uint32_t st) {
                constexpr int NB = decltype(nb)::value;
                const uint32_t key0 = (wk * steps + st) * 16;  // in the tile
                const uint32_t first = first0 + st * 16;       // in the cache
                float s[2 * NB][4] = {};
                {
                    // (one block: two chains of accumulators, half the latency of eight dependent MMAs)
                    float s2[2][4] = {};
                    const uint32_t krow = kbase + (key0 + (lane >> 4) * 8 + (lane & 7)) * 128;
#pragma unroll
                    for (int kc = 0; kc < D / 16; ++kc) {
                        uint32_t qa[4];
                        ldmatrix_x4(qa[0], qa[1], qa[2], qa[3], q_lane + q_off[kc & 3] + (kc >> 2) * 128);
#pragma unroll
                        for (int n = 0; n < NB; ++n) {
                            uint32_t b0, b1, b2, b3;
                            ldmatrix_x4(b0, b1, b2, b3, krow + k_off[kc & 3] + (kc >> 2) * kPartBytes + n * 2048);
                            mma_16816<BF16>(NB == 1 && (kc & 1) ? s2[0] : s[2 * n], qa, b0, b1);
                            mma_16816<BF16>(NB == 1 && (kc & 1) ? s2[1] : s[2 * n + 1], qa, b2, b3);
                        }
                    }
                    if constexpr (NB == 1) {
#pragma unroll
                        for (int n = 0; n < 2; ++n)
#pragma unroll
                            for (int i = 0; i < 4; ++i) s[n][i] += s2[n][i];
                    }
                }
                if (st + NB >= live) {  // the keys' slot can be filled again
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bars + 8 * (slots + k_slot));
                }
                const bool tail = first + 16 * NB > cur.len;  // the last rows: what lies behind them in the cache must not matter
                if (tail) {
#pragma unroll
                    for (int n = 0; n < 2 * NB; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (first + n * 8 + (lane & 3) * 2 + (i & 1) >= cur.len) s[n][i] = -INFINITY;
                }
                if (cur.own && p.raw) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const uint32_t g = wr * 16 + half * 8 + lane / 4;
                        if (g < p.group) {
                            float* dst = p.raw + (static_cast<size_t>(cur.b) * p.n_heads + kvh * p.group + g) * p.raw_stride + first + (lane & 3) * 2;
#pragma unroll
                            for (int n = 0; n < 2 * NB; ++n)
                                if (n < 2 || first + n * 8 < cur.len)  // (the row of scores is a multiple of 16 keys long)
                                    *reinterpret_cast<float2*>(dst + n * 8) = make_float2(s[n][2 * half] * p.scale_log2, s[n][2 * half + 1] * p.scale_log2);
                        }
                    }
                }
                // What the probabilities are relative to, the maximum less the lift, moves only when the maximum grew by more than 2^8: the
                // true sum normalises at the end, and probabilities stay below 2^8 (2^15 with fp16's lift).
                float mx[2];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float x = fmaxf(s[0][2 * half], s[0][2 * half + 1]);
#pragma unroll
                    for (int n = 1; n < 2 * NB; ++n) x = fmaxf(x, fmaxf(s[n][2 * half], s[n][2 * half + 1]));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
                    mx[half] = x * p.scale_log2;
                }
                constexpr float kLift = tc::kLift<BF16>;
                const bool grow0 = mx[0] > m[0] + (8.f + kLift), grow1 = mx[1] > m[1] + (8.f + kLift);
                if (__any_sync(0xffffffffu, grow0 || grow1)) {
                    const float m0 = mx[0] - kLift, m1 = mx[1] - kLift, f0 = grow0 ? tc::fast_exp2(m[0] - m0) : 1.f, f1 = grow1 ? tc::fast_exp2(m[1] - m1) : 1.f;
                    if (grow0) m[0] = m0;
                    if (grow1) m[1] = m1;
                    l[0] *= f0;
                    l[1] *= f1;
#pragma unroll
                    for (int i = 0; i < D / 8; ++i) {
                        o[i][0] *= f0;
                        o[i][1] *= f0;
                        o[i][2] *= f1;
                        o[i][3] *= f1;
                    }
                }
                const float ref[2] = {m[0] == -INFINITY ? 0.f : -m[0], m[1] == -INFINITY ? 0.f : -m[1]};
#pragma unroll
                for (int n = 0; n < 2 * NB; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        s[n][i] = tc::fast_exp2(fmaf(s[n][i], p.scale_log2, ref[i >> 1]));
                        l[i >> 1] += s[n][i];
                    }
                if (st == 0) ok = mbar_wait(bars + 8 * v_slot, v_phase);
                if (!ok) return;
                if (tail) {
                    for (uint32_t i = lane; i < NB * 16 * kParts * 8; i += 32) {
                        const uint32_t r = i / (kParts * 8), in_row = i % (kParts * 8);
                        if (first + r >= cur.len) st_shared_zero16(vbase + (in_row >> 3) * kPartBytes + (key0 + r) * 128 + ((in_row & 7) << 4));
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // in front of the copy that refills the slot
                    __syncwarp();
                }
                const uint32_t vrow = vbase + (key0 + ((lane >> 3) & 1) * 8 + (lane & 7)) * 128;
                if constexpr (RES) {
                    // P in three parts of bf16, which hold its 24 bits, or two of fp16, which hold 23 of a lifted p above 2^-2 (p above 2^-9 of the
                    // running maximum) and 2^-32 of that maximum below. A matrix instruction cuts its sum off instead of rounding it, which makes long sums
                    // small (4e-6 of them after 440 instructions): each starts from zero here and is added to the rest by an addition.
                    constexpr int kTerms = BF16 ? 3 : 2;
                    uint32_t pa[NB][kTerms][4];
#pragma unroll
                    for (int n = 0; n < NB; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            float x = s[2 * n + (i >> 1)][(i & 1) * 2], y = s[2 * n + (i >> 1)][(i & 1) * 2 + 1];
#pragma unroll
                            for (int t = 0; t < kTerms; ++t) {
                                pa[n][t][i] = BF16 ? pack_upper16(x, y) : pack2<BF16>(x, y);
                                x -= BF16 ? upper16(x) : round16<BF16>(x);
                                y -= BF16 ? upper16(y) : round16<BF16>(y);
                            }
                        }
#pragma unroll
                    for (int dc = 0; dc < D / 16; ++dc) {
                        float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int n = 0; n < NB; ++n) {
                            uint32_t b0, b1, b2, b3;
                            ldmatrix_x4_trans(b0, b1, b2, b3, vrow + v_off[dc & 3] + (dc >> 2) * kPartBytes + n * 2048);
#pragma unroll
                            for (int t = kTerms - 1; t >= 0; --t) {
                                mma_16816<BF16>(x, pa[n][t], b0, b1);
                                mma_16816<BF16>(y, pa[n][t], b2, b3);
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            o[2 * dc][i] += x[i];
                            o[2 * dc + 1][i] += y[i];
                        }
                    }
                } else {
#pragma unroll
                    for (int n = 0; n < NB; ++n) {
                        uint32_t pa[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            pa[i] = pack2<BF16>(s[2 * n + (i >> 1)][(i & 1) * 2], s[2 * n + (i >> 1)][(i & 1) * 2 + 1]);
#pragma unroll
                        for (int dc = 0; dc < D / 16; ++dc) {
                            uint32_t b0, b1, b2, b3;
                            ldmatrix_x4_trans(b0, b1, b2, b3, vrow + v_off[dc & 3] + (dc >> 2) * kPartBytes + n * 2048);
                            mma_16816<BF16>(o[2 * dc], pa, b0, b1);
                            mma_16816<BF16>(o[2 * dc + 1], pa, b2, b3);
                        }
                    }
                }
            };
            if (steps == 1) {
                if (live && ok) blocks(std::integral_constant<int, 1>{}, 0);
            } else {  // (a second block behind the last keys is masked like the rest of a last block)
#pragma unroll 1
                for (uint32_t st = 0; st < live && ok; st += 2) blocks(std::integral_constant<int, 2>{}, st);
            }
            if (live == 0 && ok) ok = mbar_wait(bars + 8 * v_slot, v_phase);  // (every consumer follows every phase of every slot)
            if (!ok) {
                if (p.status) atomicOr(p.status, ATTN_STATUS_WAIT_TIMEOUT);
                break;
            }
            __syncwarp();
            if (lane == 0) {
                if (live == 0) mbar_arrive(bars + 8 * (slots + k_slot));
                mbar_arrive(bars + 8 * (slots + v_slot));
            }
            if (cur.tile + 1 == cur.tiles || cur.unit + (cur.own ? 1 : p.prefix_weight) >= u1) {
                // ---- the run's piece: normalised sum and log-sum-exp (log2 units) of this warp's rows and keys
                const size_t rec = (static_cast<size_t>(cta + cur.seg) * sh.ts + wk) * sh.hpc + hs;
                float* po = cur.own ? p.part_own : p.part_pre;
                float* pl = cur.own ? p.lse_own : p.lse_pre;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float sum = l[half];
                    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                    const float inv = sum == 0.f ? 0.f : 1.f / sum;  // (a sum of NaN stays one)
                    const uint32_t r = wr * 16 + half * 8 + lane / 4;
                    const bool there = cur.own ? r < p.group : cur.rb * sh.wm * 16 + r < p.batch * p.group;
                    if (there) {
                        float* dst = po + (rec * sh.rec_rows + r) * D + (lane & 3) * 2;
#pragma unroll
                        for (int i = 0; i < D / 8; ++i)
                            *reinterpret_cast<float2*>(dst + i * 8) = make_float2(o[i][2 * half] * inv, o[i][2 * half + 1] * inv);
                        if ((lane & 3) == 0) pl[rec * sh.rec_rows + r] = sum == 0.f ? -INFINITY : (m[half] + tc::kLift<BF16>) + __log2f(sum * tc::kUnlift<BF16>);
                    }
                }
                fresh = true;
            }
            advance(cur);
        }
    }
}

// The prefix kernel, and the split pass `own` (own rows only, own_smem bytes of shared memory for each of its CTAs) on further CTAs of the same launch.
int launch_shared_prefix(const SharedPrefixParams& p, const SharedParams& own, const CUtensorMap& tm_own_k, const CUtensorMap& tm_own_v, size_t own_smem,
                         cudaStream_t stream);

}  // namespace b200
