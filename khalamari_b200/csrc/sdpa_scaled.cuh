// Map / direct attention kernels over scaled 8-bit pages (scaled_kv.cuh), for tasks of up to 32 Q rows.
//
//   s_t = scale * 2^eK_t * (q . cK_t)      p_t = exp(s_t - m)      out = sum_t p_t 2^eV_t cV_t / sum_t p_t
//
// with codes c and row exponents e. Codes are exact f16 values, so both products run as m16n8k16 f16 MMAs on codes
// with f32 accumulators, and the row scales enter where a token is one number instead of D: 2^eK multiplies the
// token's score, 2^eV its probability. The KV tokens are the M dimension (16 a tile), the Q rows the N dimension
// (NQ n-tiles of 8): S^T = K Q^T, O^T += V^T P^T.
//
// Two running references per Q row, both raised lazily (only when exceeded by 2^8): m for the scores, which the sum
// is relative to, and r for score + eV (all in the log2 domain), which the value weights w_t = 2^(s_t + eV_t - r) are
// relative to. A weight is then at most 2^8 whatever the V scales are. Rounding it to f16 costs at most 2^-11 of the term it
// multiplies for weights from 2^-14 on, and 2^-25 for smaller ones (those below 2^-25 vanish, while the sum counts their
// probability): n tokens far below a dominant one lose at most n 2^-25 of its term, n being the tokens of one warp's share.
// One reference for both would push the weights of tokens with small V rows out of f16's range. The output is
// O * 2^(r - m) / l.
//
// K and V codes of a 16-token tile arrive by TMA (128-byte swizzle), its scale bytes by a small bulk copy, on one
// mbarrier per slot of a ring that belongs to one warp, or to a pair of warps that work on neighbouring KV heads of the
// same tokens (HP = 2: their rows are neighbours in the page, so one copy brings 4 KiB of K and 4 KiB of V instead of
// 2 + 2; at 2 KiB HBM gives about 5 of its 6.5 TB/s). Each lane then reads exactly the bytes its own MMA fragments are
// made of: a sum over the head dimension does not care about order, so lane (g, t) of the 8 x 4 lane grid takes 16-byte
// chunks 2t and 2t + 1 of a 128-byte line of K rows g and g + 8, four consecutive codes standing in for the fragment's
// index pairs (2t, 2t + 1) and (2t + 8, 2t + 9), with Q read in the same order; and 16-byte column g of V rows 2t,
// 2t + 1, 2t + 8, 2t + 9, which are the fragment's tokens. Under the swizzle both patterns touch every bank once.
//
// Work is divided in two ways. In both a CTA gets one contiguous run of work items (template x KV head x Q-head range;
// slices of the same rows, a chain, are neighbours), balanced by KV tokens: the run may begin and
// end inside a template (see scaled_cut).
//  - sdpa_scaled_stream_kernel: the run's tiles are cut into one contiguous share per warp, whatever items they belong
//    to, and a warp's copies run on across items. A warp that holds all tiles of a chain publishes it by itself; a
//    chain that spans warps is merged once, at the end, by the warp that holds its start, from what the others parked
//    in shared memory. No block barrier between a pass's first tile and its last.
//  - sdpa_scaled_chain_kernel: all warps share one chain after the other and merge at each chain's end: for states too
//    wide to park one for every warp beside the staging ring.
//
// What bounds them: at head_dim 128 the copies alone would take 107 us for 64 decode sequences of 1,024-8,192 tokens (64 / 8
// heads, 604 MB of codes and scales), the step takes 135-140 us with int8 codes (4.3-4.5 TB/s) and 125-130 us with E4M3
// (4.7 TB/s), its reduce included: 440 warp instructions per 16-token int8 tile and head, which 12 warps do not hide
// altogether. 16 warps with two slots each took 148 us, 8 warps 160. At head_dim 256, 24 rows (32 sequences of four verify
// tokens, 24 / 4 heads, 1.35 GB): 500 us, 2.7 TB/s; 192 accumulator registers a thread leave two warps a scheduler, which
// wait for fixed latencies. One sequence of 524,288 tokens (16 / 2 heads, 256): 117-120 us, 4.5 TB/s, by the same 8 warps.
#pragma once

#include "scaled_kv.cuh"
#include "sdpa_map.cuh"

namespace kh {

// A row's running maximum before anything was seen: far below any score, and finite, so that differences need no guard.
constexpr float kScaledNothing = -3.0e38f;

// D: head dimension. NQ: n-tiles of 8 Q rows an item holds. W: warps. HP: warps (neighbouring KV heads) that share a
// copy. STREAM: which of the two kernels.
template <int D, int NQ, int W, int HP, bool STREAM>
struct ScaledGeometry {
    static_assert(D == 128 || D == 256, "head_dim 128 or 256");
    static_assert(HP == 1 || (STREAM && D == 128 && W % 2 == 0), "pairs of warps: stream kernel at head_dim 128");
    static constexpr int kThreads = W * 32;
    static constexpr int kUnits = W / HP;
    static constexpr int kTileTokens = 16;
    static constexpr int kRows = 8 * NQ;
    static constexpr int kItems = 128;                            // items of one pass at most
    static constexpr int kSlotBytes = 2 * kTileTokens * D * HP;    // K and V codes of a tile
    static constexpr int kScaleBytes = 32 * HP;                    // and its scale bytes
    static constexpr int kRowFloats = D + 4;                       // a parked or merged row
    static constexpr int kInfoBytes = kUnits * 64 * 8;             // tile numbers of two 32-tile windows
    static constexpr int kItemBytes = kItems * 64 + (kItems + 2) * 4 + 128;
    // stream: a parked state (rows, then m, r, l per row) for every warp
    static constexpr int kParkBytes = STREAM ? W * kRows * (kRowFloats + 3) * 4 : 0;
    // chain: Q fragments (one 8-byte pair per lane and k-step), every warp's row statistics and the merged ones
    static constexpr int kQBytes = STREAM ? 0 : NQ * (D / 16) * 32 * 8;
    static constexpr int kStatBytes = STREAM ? 0 : W * kRows * 12 + kRows * 12;
    static constexpr int kMergeBytes = STREAM ? 0 : W * 8 * kRowFloats * 4;  // one n-tile of every warp, over the ring
    static constexpr int kFixedBytes = kParkBytes + kQBytes + kStatBytes + kInfoBytes + kItemBytes + 128 + 1024;
    static constexpr int kSmemLimit = 227 * 1024;
    static constexpr int kSlotsFit = (kSmemLimit - kFixedBytes) / (kUnits * (kSlotBytes + kScaleBytes + 16));
    static constexpr int kSlots = kSlotsFit > 4 ? 4 : kSlotsFit;
    static constexpr int kRingBytes = kUnits * kSlots * kSlotBytes;
    static constexpr int kBigBytes = kRingBytes > kMergeBytes ? kRingBytes : kMergeBytes;
    static constexpr int kBarBytes = kUnits * kSlots * 16;         // full and empty barriers
    static constexpr int kSmemBytes = kBigBytes + kUnits * kSlots * kScaleBytes + kBarBytes + kFixedBytes;
    static_assert(kSlots >= 2, "staging ring too small");
    static_assert(kSmemBytes <= kSmemLimit, "shared memory");
    static_assert(kParkBytes % 16 == 0 && kQBytes % 16 == 0 && kBigBytes % 1024 == 0, "alignment");
};

// A work item: one map task template (or a part of one) x KV head x Q-head range; at most kRows Q rows.
struct ScaledItem {
    uint32_t tmpl, cell;         // cell = KV head x Q-head range; with HP = 2 the first of two
    uint32_t range;              // Q range index: items of equal range and cell are slices of the same rows
    uint32_t tok_begin, num_toks;
    uint32_t kv_begin, kv_end;   // clipped to what some row sees, and to the CTA's part of the template
    uint32_t all_begin, all_end; // tokens that every row sees
    uint32_t req_slot;
    uint32_t active;
    uint32_t chain;              // index (in the pass) of the chain's first item
    uint32_t length;             // at a chain's first item: items of the chain,
    uint32_t slot;               // template index whose partial the chain's part in this CTA is published as, and the
    uint32_t empties;            // number of template indices behind it that are published as empty
};
static_assert(sizeof(ScaledItem) <= 64, "item size");

// Q rows of an item, for the lanes that stage, mask and publish them.
struct ScaledRows {
    uint32_t head_begin, num_heads, tok_begin, num_toks, heads_per_task;

    __device__ __forceinline__ ScaledRows(const MapParams& p, const ScaledItem& it, uint32_t pair = 0) {
        const uint32_t cell = it.cell + pair;
        const uint32_t skipped = (cell % p.head_ranges) * p.heads_per_task;
        head_begin = cell / p.head_ranges * p.group + skipped;
        num_heads = min(p.heads_per_task, p.group - skipped);
        tok_begin = it.tok_begin;
        num_toks = it.num_toks;
        heads_per_task = p.heads_per_task;
    }
    __device__ __forceinline__ uint32_t token(uint32_t row) const { return row / heads_per_task; }  // of the range
    __device__ __forceinline__ uint32_t head(uint32_t row) const { return head_begin + row % heads_per_task; }
    __device__ __forceinline__ bool valid(uint32_t row) const {
        return token(row) < num_toks && row % heads_per_task < num_heads;
    }
};

// A wait of a whole warp: the same answer in every lane.
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag, const MapParams& p) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, p));
}

// One lane of a converged warp, the same one every time. Tensor-core instructions and bulk copies issued under it need no
// handling of operands that differ between lanes, which under `lane == 0` costs each of them about a hundred cycles.
__device__ __forceinline__ bool elect_one() {
    uint32_t elected;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(elected));
    return elected != 0;
}

__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, int32_t row, int32_t page, uint32_t bar,
                                            uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint "
        "[%0], [%1, {%2, %3, %2, %2, %4}], [%5], %6;"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(row), "r"(page), "r"(bar), "l"(policy)
        : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// Visible range of the range's token `tok`, cut to the template's [kv_begin, kv_end).
__device__ __forceinline__ void scaled_visible(const MapParams& p, uint32_t tok_begin, uint32_t tok, uint32_t kv_begin,
                                               uint32_t kv_end, uint32_t& lo, uint32_t& hi) {
    lo = kv_begin;
    hi = kv_end;
    if (p.visible != nullptr) {
        lo = max(lo, p.visible[(uint64_t(tok_begin) + tok) * 2]);
        hi = min(hi, p.visible[(uint64_t(tok_begin) + tok) * 2 + 1]);
    }
}

// A cut between two CTAs' runs: template `tmpl` (of one cell group's list), its tile `tile`. `interior`: the cut lies
// inside the chain of templates [chain_begin, chain_end), whose parts are published as partials
// chain_begin, chain_begin + 1, ..; `ordinal` counts the parts before this cut.
struct ScaledCut {
    uint32_t tmpl, tile, interior, ordinal, chain_begin, chain_end;
};

// Costs of a cell group's templates: prefix[i] = sum over earlier templates of (16-token tiles + kScaledOverhead).
constexpr uint32_t kScaledOverhead = 3;

__device__ __forceinline__ uint32_t scaled_cost(uint32_t range, uint32_t kv_begin, uint32_t kv_end) {
    return (range == 0xffffffffu || kv_end <= kv_begin ? 0u : (kv_end + 15) / 16 - kv_begin / 16) + kScaledOverhead;
}

// Cut number `cut` of `cuts` equal shares of `groups` cell groups' costs, local to group `group` (called by a whole warp,
// for a cut that lies in the group). A cut inside a chain may fall on any tile when the chain has at least as many
// templates as the cuts make parts of it, since every part needs a partial of its own; else it moves to the nearer
// end of its template. `splittable`: chains may be cut at all.
__device__ __forceinline__ ScaledCut scaled_cut(const uint32_t* prefix, const uint32_t* ranges, uint32_t templates, uint64_t groups,
                                                uint64_t group, uint64_t cut, uint64_t cuts, bool splittable, uint32_t max_chain,
                                                uint32_t lane) {
    const uint64_t per_group = prefix[templates], total = per_group * groups;
    const uint32_t x = uint32_t(total * cut / cuts - group * per_group);
    ScaledCut c{templates, 0, 0, 0, 0, 0};
    if (x >= per_group) return c;
    uint32_t lo = 0, hi = templates;  // the last template that starts at or before x
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (prefix[mid] <= x) lo = mid;
        else hi = mid;
    }
    const uint32_t offset = x - prefix[lo], tiles = prefix[lo + 1] - prefix[lo] - kScaledOverhead;
    c.tmpl = lo;
    c.tile = offset > kScaledOverhead ? offset - kScaledOverhead : 0;
    // the chain around the template
    const uint32_t range = ranges[lo];
    uint32_t begin = lo, end = lo + 1;
    while (begin > 0) {
        const bool same = lane < begin && ranges[begin - 1 - lane] == range;
        const uint32_t differ = __ballot_sync(0xffffffffu, !same);
        const uint32_t run = differ ? uint32_t(__ffs(int(differ))) - 1 : 32;
        begin -= run;
        if (run < 32) break;
    }
    while (end < templates) {
        const bool same = end + lane < templates && ranges[end + lane] == range;
        const uint32_t differ = __ballot_sync(0xffffffffu, !same);
        const uint32_t run = differ ? uint32_t(__ffs(int(differ))) - 1 : 32;
        end += run;
        if (run < 32) break;
    }
    // Cuts inside the chain: positions behind its first tile (a cut in the overhead of the first template is a cut at
    // the chain's start) and before its end.
    const uint64_t from = group * per_group + prefix[begin] + kScaledOverhead + 1, to = group * per_group + prefix[end];
    const uint64_t first = (from * cuts + total - 1) / total, last = (to * cuts + total - 1) / total - 1;
    const bool inside = cut >= first && cut <= last;
    if (inside && splittable && total / cuts >= 8 && end - begin >= last - first + 2 && end - begin <= max_chain) {
        c.interior = 1;
        c.ordinal = uint32_t(cut - first) + 1;
        c.chain_begin = begin;
        c.chain_end = end;
    } else {
        if (c.tile * 2 > tiles) ++c.tmpl;
        c.tile = 0;
    }
    return c;
}

// This CTA's run: a range of templates, its first and last possibly in part, of one cell group.
struct ScaledRun {
    ScaledCut begin, end;
    uint32_t group;
    uint32_t templates;  // of the run
};

// Item `index` of a run, cell-major, with the early-return rules of decode_task (sdpa_map.cuh).
template <int HP>
__device__ __forceinline__ ScaledItem scaled_item(const MapParams& p, const ActiveCounts& a, const ScaledRun& run, uint32_t index) {
    ScaledItem it;
    it.active = 0;
    it.kv_begin = it.kv_end = it.all_begin = it.all_end = 0;
    it.tok_begin = it.num_toks = it.req_slot = 0;
    it.chain = it.length = it.empties = 0;
    it.tmpl = run.begin.tmpl + index;
    it.slot = it.tmpl;
    it.cell = run.group * HP;
    it.range = p.templates[uint64_t(it.tmpl) * 3];
    const uint32_t kv_begin = p.templates[uint64_t(it.tmpl) * 3 + 1], kv_end = p.templates[uint64_t(it.tmpl) * 3 + 2];
    if (p.q_ranges == nullptr) {
        if (it.range >= a.tokens) return it;
        it.tok_begin = it.range;
        it.num_toks = 1;
    } else {
        if (it.range >= a.q_tiles) return it;
        const uint32_t begin = p.q_ranges[it.range * 2], end = p.q_ranges[it.range * 2 + 1];
        if (begin >= a.tokens || end > a.tokens || end <= begin) return it;
        it.tok_begin = begin;
        it.num_toks = min(end - begin, p.max_q_tokens);
    }
    it.req_slot = p.req_slots[it.tok_begin];
    if (it.req_slot >= p.num_req_slots ||
        (kv_end > kv_begin &&
         (uint64_t(kv_end) + p.tokens_per_page - 1) / p.tokens_per_page > p.pages_per_request_layer)) {
        atomicOr(p.status, kStatusMetadataOutOfRange);  // the task is dropped, as in decode_task
        return it;
    }
    it.active = 1;
    uint32_t any_lo = 0xffffffffu, any_hi = 0, all_lo = 0, all_hi = 0xffffffffu;
    for (uint32_t tok = 0; tok < it.num_toks; ++tok) {
        uint32_t lo, hi;
        scaled_visible(p, it.tok_begin, tok, kv_begin, kv_end, lo, hi);
        all_lo = max(all_lo, lo);
        all_hi = min(all_hi, hi);
        if (hi > lo) {
            any_lo = min(any_lo, lo);
            any_hi = max(any_hi, hi);
        }
    }
    // the CTA's part of a template that a cut divides
    if (index == 0 && run.begin.tile > 0) any_lo = max(any_lo, (kv_begin / 16 + run.begin.tile) * 16);
    if (it.tmpl == run.end.tmpl) any_hi = min(any_hi, (kv_begin / 16 + run.end.tile) * 16);
    if (any_hi > any_lo) {
        it.kv_begin = any_lo;
        it.kv_end = any_hi;
    }
    it.all_begin = all_lo;
    it.all_end = all_hi;
    return it;
}

// Warp 0, after the items of a pass have been written: chains, the partials they are published as, and the prefix sum of
// the items' tiles. A pass ends with the last whole chain that fits it (ONE_CHAIN: with the first); returns its items.
template <bool ONE_CHAIN>
__device__ __forceinline__ uint32_t scaled_chains(const MapParams& p, const ScaledRun& run, ScaledItem* items, uint32_t* cum, uint32_t count,
                                                  bool more, uint32_t lane) {
    // an item continues the one before it when it is another slice of the same Q rows whose state can be carried on
    auto continues = [&](uint32_t i) {
        return i > 0 && p.direct == 0 && items[i].active && items[i - 1].active && items[i].range == items[i - 1].range;
    };
    uint32_t chain = 0, kept = count;
    for (uint32_t base = 0; base < count; base += 32) {
        const uint32_t i = base + lane;
        const uint32_t starters = __ballot_sync(0xffffffffu, i < count && !continues(i));
        if (ONE_CHAIN) {
            const uint32_t second = base == 0 ? starters & ~1u : starters;
            if (second != 0 && kept == count) kept = base + __ffs(int(second)) - 1;
        }
        const uint32_t mine = starters & (0xffffffffu >> (31 - lane));  // chain starts up to this lane
        const uint32_t my_chain = mine != 0 ? base + 31 - __clz(int(mine)) : chain;
        if (i < count) items[i].chain = my_chain;
        chain = __shfl_sync(0xffffffffu, my_chain, 31);
    }
    // (`chain` is now the last chain's first item: left for the next pass when the run goes on and it is not the only one)
    if (!ONE_CHAIN && more && chain > 0) kept = chain;
    __syncwarp();
    uint32_t total = 0;
    for (uint32_t base = 0; base < kept; base += 32) {
        const uint32_t i = base + lane;
        uint32_t tiles = 0;
        if (i < kept && items[i].kv_end > items[i].kv_begin) tiles = (items[i].kv_end + 15) / 16 - items[i].kv_begin / 16;
        uint32_t scan = tiles;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, scan, d);
            if (lane >= uint32_t(d)) scan += v;
        }
        if (i < kept) {
            cum[i] = total + scan - tiles;
            if (items[i].chain == i) {
                uint32_t length = 1;
                while (i + length < kept && items[i + length].chain == i) ++length;
                const uint32_t first_tmpl = items[i].tmpl, last_tmpl = items[i + length - 1].tmpl;
                items[i].length = length;
                // whole chains, and parts that begin and end with a template: the first template's partial
                uint32_t slot = first_tmpl, empties = length - 1;
                if (run.begin.interior && first_tmpl >= run.begin.chain_begin && first_tmpl < run.begin.chain_end) {
                    slot = run.begin.chain_begin + run.begin.ordinal;
                    empties = run.begin.chain_end - slot - 1;  // (none where the chain goes on behind the run: below)
                }
                if (run.end.interior && last_tmpl >= run.end.chain_begin && last_tmpl < run.end.chain_end) empties = 0;
                items[i].slot = slot;
                items[i].empties = empties;
            }
        }
        total += __shfl_sync(0xffffffffu, scan, 31);
    }
    if (lane == 0) cum[kept] = total;
    return kept;
}

// The copies of one unit's tiles [begin, end) of a pass. Warp 0 of the unit issues; `info` keeps the tiles' numbers
// (two 32-tile windows: a tile is consumed at most kSlots tiles after it was issued). Slots and barrier phases follow a
// running count of the unit's tiles.
template <typename G, int D, int HP>
struct ScaledFetch {
    const MapParams& p;
    const CUtensorMap* map;
    const ScaledItem* items;
    const uint32_t* cum;
    uint2* info;            // [64]: {item | chain << 8 | 0x80000000 where every row sees the whole tile, first token}
    volatile uint32_t* abort_flag;
    uint64_t policy;
    uint32_t ring, scales, full_bar, empty_bar;  // shared-memory addresses of the unit's slots
    uint32_t count, begin, end;
    uint32_t lane, page_shift;
    uint32_t issued;        // running count of the unit's tiles
    uint32_t slot, phase;   // of the next one
    // lane i: tile (window base + i)
    uint32_t page0, page1, row0;  // pages of its 8-token halves, first row in the page's K plane

    __device__ __forceinline__ uint32_t page_of(uint64_t table, uint32_t token) {
        uint32_t page = p.page_ids[table + (token >> page_shift)];
        if (page >= p.pool_pages) {  // nothing outside the pool is read: the output is then meaningless, and reported
            atomicOr(p.status, kStatusPageOutOfPool);
            page = 0;
        }
        return page;
    }

    __device__ __forceinline__ void load_window(uint32_t base) {
        const uint32_t x = base + lane;
        if (x >= end) return;
        uint32_t lo = 0, hi = count;
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (cum[mid] <= x) lo = mid;
            else hi = mid;
        }
        const ScaledItem& it = items[lo];
        const uint32_t tok = (it.kv_begin / 16 + x - cum[lo]) * 16;
        const bool inside = tok >= it.all_begin && tok >= it.kv_begin && tok + 16 <= it.all_end && tok + 16 <= it.kv_end;
        info[(x - begin) & 63] = make_uint2(lo | (it.chain << 8) | (inside ? 0x80000000u : 0u), tok);
        const uint64_t table = (uint64_t(it.req_slot) * p.num_gqa_layers + p.layer_index) * p.pages_per_request_layer;
        // A half that holds no token of the item is not looked up (its page may not exist): the other one's page stands in,
        // and its tokens are masked.
        const bool low = tok + 8 > it.kv_begin, high = tok + 8 < it.kv_end;
        page0 = page_of(table, low ? tok : tok + 8);
        page1 = page0;
        if (page_shift == 3 && low && high) page1 = page_of(table, tok + 8);
        row0 = ((it.cell / p.head_ranges) << page_shift) + ((tok >> 4 << 4) & (p.tokens_per_page - 1));
    }

    // The next tile x = begin, begin + 1, .. into its slot; false when a wait ran out.
    __device__ __forceinline__ bool issue(uint32_t x) {
        if (x >= end) return true;
        const uint32_t i = (x - begin) & 31;
        if (i == 0) {
            load_window(x);
            __syncwarp();  // lane 0's arrival below publishes every lane's tile numbers to the unit's other warp
        }
        const uint32_t first_page = __shfl_sync(0xffffffffu, page0, int(i)), row = __shfl_sync(0xffffffffu, row0, int(i));
        const uint32_t second_page = __shfl_sync(0xffffffffu, page1, int(i));
        if (!mbar_wait_warp(empty_bar + 8 * slot, phase ^ 1, abort_flag, p)) return false;
        if (elect_one()) {
            const uint32_t bar = full_bar + 8 * slot, dst = ring + slot * G::kSlotBytes, sdst = scales + slot * G::kScaleBytes;
            const uint32_t P = p.tokens_per_page;
            mbar_arrive_expect_tx(bar, G::kSlotBytes + G::kScaleBytes);
            // scale bytes of the first head's K rows
            const uint8_t* s0 = p.kv_pages + uint64_t(first_page) * p.page_bytes + uint64_t((p.num_kv_heads * 2) << page_shift) * D +
                                ((row >> page_shift << page_shift) * 2) + (row & (P - 1));
            tma_load_5d(dst, map, int32_t(row), int32_t(first_page), bar, policy);
            if (page_shift == 3) {  // two 8-token pages
                const uint8_t* s1 = s0 + (int64_t(second_page) - int64_t(first_page)) * p.page_bytes;
                tma_load_5d(dst + G::kSlotBytes / 2, map, int32_t(row), int32_t(second_page), bar, policy);
                bulk_load(sdst, s0, G::kScaleBytes / 2, bar);
                bulk_load(sdst + G::kScaleBytes / 2, s1, G::kScaleBytes / 2, bar);
            } else if (page_shift == 4) {
                bulk_load(sdst, s0, G::kScaleBytes, bar);
            } else {  // half of a 32-token page: its K and its V bytes
                bulk_load(sdst, s0, 16, bar);
                bulk_load(sdst + 16, s0 + P, 16, bar);
            }
        }
        __syncwarp();
        ++issued;
        if (++slot == uint32_t(G::kSlots)) {
            slot = 0;
            phase ^= 1;
        }
        return true;
    }
};

// Abort path only: copies already issued may still be landing; wait (bounded) for each before the CTA may retire.
template <typename G, typename F>
__device__ __forceinline__ void scaled_drain(const MapParams& p, const F& fetch, bool issues, volatile uint32_t* abort_flag, uint32_t lane) {
    if (*abort_flag == 0 || !issues || lane != 0) return;
    uint32_t slot = fetch.slot, phase = fetch.phase;
    for (uint32_t back = 0; back < uint32_t(G::kSlots) && back < fetch.issued; ++back) {
        if (slot == 0) {
            slot = G::kSlots;
            phase ^= 1;
        }
        --slot;
        for (uint32_t i = 0; i < p.wait_limit; ++i) {
            if (mbar_try_wait(fetch.full_bar + 8 * slot, phase)) break;
        }
    }
}

// Where a lane finds its bytes in a slot.
template <int D, int HP>
struct ScaledLane {
    uint32_t k[2], v[2];  // K row g / g + 8, line 0, chunk 2t; V row 2t / 2t + 8, line 0, column g
    uint32_t scale[2];    // K scale byte of token g / g + 8
    uint32_t line;        // bytes between the 128-byte lines of a row (head_dim 256)
    uint32_t v_scale;     // bytes from a token's K scale byte to its V scale byte

    __device__ __forceinline__ ScaledLane(uint32_t tokens_per_page, uint32_t pair, uint32_t lane) {
        const uint32_t g = lane >> 2, t = lane & 3;
        const uint32_t held = min(tokens_per_page, 16u);  // tokens of a head in one copy
        const uint32_t rows = held * HP;                  // rows of one plane and line of a copy
        line = rows * 128;
        const uint32_t plane = line * (D / 128);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t box = held == 8 ? h * 2 * plane : 0, first = pair * held + (held == 8 ? 0 : 8 * h);
            k[h] = box + (first + g) * 128 + (((2 * t) ^ g) << 4);
            v[h] = box + plane + (first + 2 * t) * 128 + ((g ^ (2 * t)) << 4);
            scale[h] = held == 8 ? (h * HP + pair) * 16 + g : pair * 32 + 8 * h + g;
        }
        v_scale = held;
    }
};

// Q fragments of n-tile n for one lane: row n * 8 + g, elements 128 (c / 2) + 32 t + 16 (c % 2) + (0 .. 15)
// as f16 pairs, `put(step, pair)`.
// bf16 rows are scaled by a power of two so that their largest element lies in [2^8, 2^9): exact in f16 down to 2^-22 of
// that element, and no bf16 value overflows. Returns the factor from the row's dot products to log2-domain scores; NaN for a
// row that is not finite, whose softmax is NaN wherever it sees a token (left to the scores, a row of -inf would look like
// one that sees nothing).
template <typename T, int D, typename Put>
__device__ __forceinline__ float scaled_load_q(const MapParams& p, const ScaledRows& rows, uint32_t n, uint32_t lane, Put put) {
    constexpr int KC = D / 64;
    const uint32_t row = n * 8 + (lane >> 2), t = lane & 3;
    uint4 raw[KC][2];
    if (rows.valid(row)) {
        const uint64_t q_row = (uint64_t(rows.tok_begin) + rows.token(row)) * p.num_q_heads + rows.head(row);
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + q_row * D);
#pragma unroll
        for (int c = 0; c < KC; ++c) {
            raw[c][0] = src[c / 2 * 16 + t * 4 + c % 2 * 2];
            raw[c][1] = src[c / 2 * 16 + t * 4 + c % 2 * 2 + 1];
        }
    } else {
#pragma unroll
        for (int c = 0; c < KC; ++c) raw[c][0] = raw[c][1] = make_uint4(0, 0, 0, 0);
    }
    float factor = p.scale_log2e, up = 1.0f;
    uint32_t most = 0;  // the row's largest magnitude bits (ordered as integers)
#pragma unroll
    for (int c = 0; c < KC; ++c) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            most = __vmaxu2(most, __vmaxu2(__vmaxu2(raw[c][h].x & 0x7fff7fffu, raw[c][h].y & 0x7fff7fffu),
                                           __vmaxu2(raw[c][h].z & 0x7fff7fffu, raw[c][h].w & 0x7fff7fffu)));
        }
    }
    most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, 2));
    most = max(most & 0xffffu, most >> 16);
    constexpr uint32_t kInfinity = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    if (most >= kInfinity) {
        factor = __uint_as_float(0x7fc00000u);  // a NaN or an infinity: all scores of the row are NaN or infinite
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        // of the largest element, biased (rows below 2^-111 stay below 2^8, so that the factor is no subnormal)
        const int exponent = max(int(most >> 7), 16);
        up = __uint_as_float(uint32_t(262 - exponent) << 23);  // 2^(8 - k), k = exponent - 127
        factor = p.scale_log2e * __uint_as_float(uint32_t(exponent - 8) << 23);
    }
#pragma unroll
    for (int c = 0; c < KC; ++c) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const uint4 v = raw[c][w / 2];
            uint2 pair = w % 2 == 0 ? make_uint2(v.x, v.y) : make_uint2(v.z, v.w);
            if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                const float2 x = unpack2<__nv_bfloat16>(pair.x), y = unpack2<__nv_bfloat16>(pair.y);
                pair = make_uint2(pack2<__half>(x.x * up, x.y * up), pack2<__half>(y.x * up, y.y * up));
            }
            put(c * 4 + w, pair);
        }
    }
    return factor;
}

// Running state of NQ n-tiles. Lane (g, t): accumulators of O^T for rows 2t, 2t + 1 and head-dim elements
// 128 c + 16 g + 2 j, + 1 (acc[n][8 c + j]); references and partial sums (over the lane's tokens) of the same rows.
template <int D, int NQ>
struct ScaledState {
    float acc[NQ][D / 16][4];
    float m[NQ][2], r[NQ][2], l[NQ][2], factor[NQ][2];

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
#pragma unroll
            for (int j = 0; j < D / 16; ++j) acc[n][j][0] = acc[n][j][1] = acc[n][j][2] = acc[n][j][3] = 0.0f;
            m[n][0] = m[n][1] = r[n][0] = r[n][1] = kScaledNothing;
            l[n][0] = l[n][1] = 0.0f;
        }
    }
    // Sums over the lanes that share a row.
    __device__ __forceinline__ void finish_sums() {
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int d = 4; d <= 16; d <<= 1) l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], d);
            }
        }
    }
};

// A tile of 16 tokens into the state. `slot`: its codes, `scales`: its scale bytes, `info`: its numbers (ScaledFetch).
// q(n, step): Q fragment.
template <int CODE, int D, int NQ, int HP, typename Q>
__device__ __forceinline__ void scaled_tile(const MapParams& p, ScaledState<D, NQ>& st, uint8_t* slot, const uint8_t* scales, uint2 info,
                                            const ScaledItem* items, uint32_t pair, const ScaledLane<D, HP>& at, uint32_t lane, Q q) {
    constexpr int KC = D / 64, VG = D / 128;
    constexpr int KA = NQ == 1 ? 2 : 1;  // accumulators of a score tile: one chain of MMAs alone would wait on itself
    constexpr float kMost = 256.0f;      // a reference is raised when a weight would exceed this
    const uint32_t g = lane >> 2, t = lane & 3;
    float k_scale[2], v_log[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        k_scale[h] = scale_of_byte(scales[at.scale[h]]);
        // b - 127 through the mantissa of 2^23 + b
        v_log[h] = __uint_as_float(0x4b000000u | scales[at.scale[h] + at.v_scale]) - 8388735.0f;
    }

    // ---- S^T = K Q^T
    float s[NQ][4], odd[KA == 2 ? 4 : 1];
#pragma unroll
    for (int n = 0; n < NQ; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
    if constexpr (KA == 2) odd[0] = odd[1] = odd[2] = odd[3] = 0.0f;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
        uint32_t w0[4], w1[4];
        const uint32_t line = c / 2 * at.line, flip = c % 2 * 16;
        const uint4 k0 = *reinterpret_cast<const uint4*>(slot + line + (at.k[0] ^ flip));
        const uint4 k1 = *reinterpret_cast<const uint4*>(slot + line + (at.k[1] ^ flip));
        w0[0] = k0.x, w0[1] = k0.y, w0[2] = k0.z, w0[3] = k0.w;
        w1[0] = k1.x, w1[1] = k1.y, w1[2] = k1.z, w1[3] = k1.w;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            uint32_t frag[4];
            codes4_to_half<CODE>(w0[w], frag[0], frag[2]);
            codes4_to_half<CODE>(w1[w], frag[1], frag[3]);
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                const uint2 b = q(n, c * 4 + w);
                if constexpr (KA == 2) {
                    if (w & 1) mma_16816<__half>(odd, frag, b.x, b.y);
                    else mma_16816<__half>(s[n], frag, b.x, b.y);
                } else {
                    mma_16816<__half>(s[n], frag, b.x, b.y);
                }
            }
        }
    }
    if constexpr (KA == 2) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[0][e] += odd[e];
    }
    // ---- scores in the log2 domain: lane (g, t) holds tokens g, g + 8 (s[0..1], s[2..3]) of rows 2t, 2t + 1
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] *= k_scale[e / 2] * st.factor[n][e % 2];
    }
    if ((info.x >> 31) == 0) {  // some row does not see all 16 tokens
        const ScaledItem& item = items[info.x & 0xffu];
        const uint32_t tok = info.y;
        const ScaledRows rows(p, item, pair);
        const uint32_t tmpl_begin = p.templates[uint64_t(item.tmpl) * 3 + 1], tmpl_end = p.templates[uint64_t(item.tmpl) * 3 + 2];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const uint32_t row = n * 8 + 2 * t + c;
                uint32_t lo = 0, hi = 0;
                if (rows.valid(row)) scaled_visible(p, rows.tok_begin, rows.token(row), tmpl_begin, tmpl_end, lo, hi);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t token = tok + 8 * h + g;
                    if (token < lo || token >= hi) s[n][2 * h + c] = -INFINITY;
                }
            }
        }
        if constexpr (CODE == kCodeE4M3) {
            // rows outside the item may hold anything, the NaN code among it, and 0 * NaN is NaN
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t token = tok + (r / 2) * 8 + 2 * t + r % 2;
                if (token < item.kv_begin || token >= item.kv_end) {
#pragma unroll
                    for (int c = 0; c < VG; ++c) {
                        *reinterpret_cast<uint4*>(slot + c * at.line + (at.v[r / 2] ^ (r % 2 * 16)) + r % 2 * 128) = make_uint4(0, 0, 0, 0);
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the slot's next copy lands after these
        }
    }
    // ---- probabilities (for the sum) and value weights, relative to the references
    float pr[NQ][4], w[NQ][4], most = 0.0f;
    auto weights = [&]() {
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                pr[n][e] = fast_exp2(s[n][e] - st.m[n][e % 2]);
                w[n][e] = fast_exp2(s[n][e] + (v_log[e / 2] - st.r[n][e % 2]));
                most = fmaxf(most, fmaxf(pr[n][e], w[n][e]));
            }
        }
    };
    weights();
    if (__any_sync(0xffffffffu, most > kMost)) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float top_s = fmaxf(kScaledNothing, fmaxf(s[n][c], s[n][2 + c]));
                float top_y = fmaxf(kScaledNothing, fmaxf(s[n][c] + v_log[0], s[n][2 + c] + v_log[1]));
#pragma unroll
                for (int d = 4; d <= 16; d <<= 1) {
                    top_s = fmaxf(top_s, __shfl_xor_sync(0xffffffffu, top_s, d));
                    top_y = fmaxf(top_y, __shfl_xor_sync(0xffffffffu, top_y, d));
                }
                if (top_s > st.m[n][c]) {
                    st.l[n][c] *= fast_exp2(st.m[n][c] - top_s);
                    st.m[n][c] = top_s;
                }
                if (top_y > st.r[n][c]) {
                    const float keep = fast_exp2(st.r[n][c] - top_y);
                    st.r[n][c] = top_y;
#pragma unroll
                    for (int j = 0; j < D / 16; ++j) {
                        st.acc[n][j][c] *= keep;
                        st.acc[n][j][2 + c] *= keep;
                    }
                }
            }
        }
        weights();
    }
    uint32_t weight[NQ][2];  // B fragments: packed pairs of rows, transposed
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        st.l[n][0] += pr[n][0] + pr[n][2];
        st.l[n][1] += pr[n][1] + pr[n][3];
        weight[n][0] = movmatrix_trans(pack2<__half>(w[n][0], w[n][1]));
        weight[n][1] = movmatrix_trans(pack2<__half>(w[n][2], w[n][3]));
    }
    // ---- O^T += V^T P^T: lane (g, t) has codes 16 g .. of tokens 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
    for (int c = 0; c < VG; ++c) {
        uint4 v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            v[r] = *reinterpret_cast<const uint4*>(slot + c * at.line + (at.v[r / 2] ^ (r % 2 * 16)) + r % 2 * 128);
        }
        const uint32_t words[4][4] = {{v[0].x, v[0].y, v[0].z, v[0].w}, {v[1].x, v[1].y, v[1].z, v[1].w},
                                      {v[2].x, v[2].y, v[2].z, v[2].w}, {v[3].x, v[3].y, v[3].z, v[3].w}};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                // bytes 2j, 2j + 1 of the four tokens: [byte][token pair]
                uint32_t frag[4];
                codes4_to_half<CODE>(__byte_perm(words[0][e], words[1][e], j == 0 ? 0x5140 : 0x7362), frag[0], frag[1]);
                codes4_to_half<CODE>(__byte_perm(words[2][e], words[3][e], j == 0 ? 0x5140 : 0x7362), frag[2], frag[3]);
#pragma unroll
                for (int n = 0; n < NQ; ++n) mma_16816<__half>(st.acc[n][c * 8 + e * 2 + j], frag, weight[n][0], weight[n][1]);
            }
        }
    }
}

// Publishes one row's statistics as the chain's partial, and the chain's empty partials.
__device__ __forceinline__ void scaled_publish_stats(const MapParams& p, const ScaledRows& rows, const ScaledItem* chain, uint32_t row,
                                                     float m, float sum) {
    const uint64_t index = (uint64_t(chain->slot) * p.num_q_heads + rows.head(row)) * p.max_q_tokens + rows.token(row);
    publish_partial_stats(p.partial_sum, p.partial_max, index, m * 0.6931471805599453f, sum);
    for (uint32_t i = 1; i <= chain->empties; ++i) {
        const uint64_t other = index + uint64_t(i) * p.num_q_heads * p.max_q_tokens;
        p.partial_sum[other] = 0.0f;
        p.partial_max[other] = -INFINITY;
    }
}

// The factor 2^(r - m) / sum from accumulators to outputs is taken in two, 2^up first: m may lag by 2^8 behind a largest score
// and V's exponents reach 2^122, while f32 ends at 2^128. An output may be 2^128 all the same (what codes of a bf16 row's
// largest value stand for): as a partial it must stay finite, so such large ones are taken 2^-20 smaller.
__device__ __forceinline__ float scaled_rise(float r, float m) { return r - m > 96.0f ? 32.0f : 0.0f; }
__device__ __forceinline__ float scaled_last_factor(float r, float m, float up, float sum) {
    const float f = sum == 0.0f ? 0.0f : fast_exp2(r - m - up) / sum;  // (a NaN sum stays NaN)
    return up > 0.0f ? f * (1.0f - 0x1p-20f) : f;
}

// Four consecutive output elements of a row into the final output, or into the chain's partial slot.
template <typename T, int D, bool DIRECT>
__device__ __forceinline__ void scaled_publish4(const MapParams& p, const ScaledRows& rows, const ScaledItem* chain, uint32_t row, uint32_t d,
                                                float4 v) {
    if constexpr (DIRECT) {
        T* const dst = static_cast<T*>(p.out) + ((uint64_t(rows.tok_begin) + rows.token(row)) * p.num_q_heads + rows.head(row)) * D + d;
        *reinterpret_cast<uint2*>(dst) = make_uint2(saturate2<T>(pack2<T>(v.x, v.y)), saturate2<T>(pack2<T>(v.z, v.w)));
    } else {
        const uint64_t index = (uint64_t(chain->slot) * p.num_q_heads + rows.head(row)) * p.max_q_tokens + rows.token(row);
        *reinterpret_cast<float4*>(p.partial_out + index * D + d) = v;
    }
}

// Prefix sums of the templates' costs, and their Q ranges. Called by all threads; `scratch`: a word per warp.
template <typename G>
__device__ __forceinline__ void scaled_prefix(const MapParams& p, uint32_t templates, uint32_t* prefix, uint32_t* ranges, uint32_t* scratch) {
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t chunk = (templates + G::kThreads - 1) / G::kThreads;
    const uint32_t first = min(tid * chunk, templates), last = min(first + chunk, templates);
    for (uint32_t i = tid; i < templates; i += G::kThreads) {
        const uint32_t range = p.templates[uint64_t(i) * 3];
        ranges[i] = range;
        prefix[i + 1] = scaled_cost(range, p.templates[uint64_t(i) * 3 + 1], p.templates[uint64_t(i) * 3 + 2]);
    }
    __syncthreads();
    uint32_t sum = 0;
    for (uint32_t i = first; i < last; ++i) sum += prefix[i + 1];
    uint32_t scan = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, scan, d);
        if (lane >= uint32_t(d)) scan += v;
    }
    if (lane == 31) scratch[warp] = scan;
    __syncthreads();
    uint32_t before = scan - sum;
    for (uint32_t w = 0; w < warp; ++w) before += scratch[w];
    for (uint32_t i = first; i < last; ++i) {
        before += prefix[i + 1];
        prefix[i + 1] = before;
    }
    if (tid == 0) prefix[0] = 0;
    __syncthreads();
}

// A CTA's share of `groups` cell groups' templates: from cut `begin` in group `first` to cut `end` in group `last`.
struct ScaledShare {
    ScaledCut begin, end;
    uint32_t first, last;  // first > last: nothing

    // The part that lies in one group.
    __device__ __forceinline__ ScaledRun run(uint32_t group, uint32_t templates) const {
        ScaledRun r;
        r.begin = group == first ? begin : ScaledCut{0, 0, 0, 0, 0, 0};
        r.end = group == last ? end : ScaledCut{templates, 0, 0, 0, 0, 0};
        r.group = group;
        const uint32_t stop = r.end.tmpl + (r.end.tile > 0 ? 1 : 0);
        r.templates = stop > r.begin.tmpl ? stop - r.begin.tmpl : 0;
        return r;
    }
};

// Called by all threads; leaves the share in shared memory (`share`). `big`: the ring, not in use yet.
template <typename G>
__device__ __forceinline__ void scaled_share(const MapParams& p, const ActiveCounts& a, uint32_t groups,
                                             uint32_t* big, uint32_t* scratch, ScaledShare* share) {
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t n = a.templates;
    const uint64_t tasks = uint64_t(n) * groups;
    const uint64_t cta = blockIdx.x, ctas = gridDim.x;
    if (tasks <= ctas || n > kBalanceMaxTemplates || (2 * n + 1) * 4 > uint32_t(G::kBigBytes)) {
        // at most one template and cell group per CTA; or so many that equal counts balance well enough
        const uint64_t from = tasks <= ctas ? min(cta, tasks) : tasks * cta / ctas;
        const uint64_t to = tasks <= ctas ? min(cta + 1, tasks) : tasks * (cta + 1) / ctas;
        if (tid == 0) {
            share->first = 1;
            share->last = 0;
            if (from < to) {
                share->first = uint32_t(from / n);
                share->last = uint32_t((to - 1) / n);
                share->begin = ScaledCut{uint32_t(from % n), 0, 0, 0, 0, 0};
                share->end = ScaledCut{uint32_t((to - 1) % n + 1), 0, 0, 0, 0, 0};
            }
        }
    } else {
        uint32_t* const prefix = big;
        uint32_t* const ranges = big + n + 1;
        const bool splittable = p.direct == 0;
        scaled_prefix<G>(p, n, prefix, ranges, scratch);
        const uint64_t per_group = prefix[n], total = per_group * groups;
        const uint64_t x0 = total * cta / ctas, x1 = total * (cta + 1) / ctas;
        const uint64_t group0 = x0 / per_group;
        uint64_t group1 = x1 / per_group;
        if (group1 > group0 && x1 == group1 * per_group) --group1;  // the share ends with a group
        if (warp < 2) {
            const ScaledCut c = scaled_cut(prefix, ranges, n, groups, warp == 0 ? group0 : group1, cta + warp, ctas, splittable,
                                           G::kItems, lane);
            if (lane == 0) *(warp == 0 ? &share->begin : &share->end) = c;
        }
        if (tid == 0) {
            share->first = uint32_t(group0);
            share->last = uint32_t(group1);
        }
        // the sums lie where the copies will land
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
}

// ------------------------------ one share of tiles per warp ------------------------------------------------------
template <typename T, int CODE, int D, int NQ, int W, int HP>
__global__ void __launch_bounds__(W * 32, 1)
sdpa_scaled_stream_kernel(const __grid_constant__ CUtensorMap kv_map, const __grid_constant__ CUtensorMap, const MapParams p) {
    using G = ScaledGeometry<D, NQ, W, HP, true>;
    constexpr int S = G::kSlots;
    constexpr int U = G::kUnits;
    constexpr int KS = D / 16;

    extern __shared__ uint8_t smem_raw[];
    uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* const park = reinterpret_cast<float*>(smem + G::kBigBytes);               // [W][rows][D + 4], then [W][3][rows]
    float* const park_stats = park + W * G::kRows * G::kRowFloats;
    uint8_t* const scale_ring = smem + G::kBigBytes + G::kParkBytes;                 // [U][S] scale bytes
    uint64_t* const bars = reinterpret_cast<uint64_t*>(scale_ring + U * S * G::kScaleBytes);  // [U][full S, empty S]
    uint2* const infos = reinterpret_cast<uint2*>(bars + U * S * 2);
    ScaledItem* const items = reinterpret_cast<ScaledItem*>(reinterpret_cast<uint8_t*>(infos) + G::kInfoBytes);
    uint32_t* const cum = reinterpret_cast<uint32_t*>(items + G::kItems);            // [kItems + 1] first tile of every item
    ScaledShare* const share = reinterpret_cast<ScaledShare*>(cum + G::kItems + 2);
    uint32_t* const pass_items = reinterpret_cast<uint32_t*>(share + 1);
    volatile uint32_t* const abort_flag = pass_items + 1;

    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t unit = warp / HP, pair = warp % HP;
    const uint32_t g = lane >> 2, t = lane & 3;
    if (tid == 0) {
        for (int i = 0; i < U * S; ++i) {
            mbar_init(smem_addr(bars + i / S * 2 * S + i % S), 1);
            mbar_init(smem_addr(bars + i / S * 2 * S + S + i % S), HP);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&kv_map)) : "memory");
    }
    __syncthreads();
    if constexpr (G::kSmemBytes + 14 * 1024 > 228 * 1024) {
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // (as in sdpa_map_kernel)
    }
    const ActiveCounts a = resolve_active(p);
    const uint32_t groups = p.num_kv_heads * p.head_ranges / HP;
    const ScaledLane<D, HP> at(p.tokens_per_page, pair, lane);
    uint8_t* const my_ring = smem + unit * (S * G::kSlotBytes);
    const uint8_t* const my_scales = scale_ring + unit * (S * G::kScaleBytes);
    uint2* const my_infos = infos + unit * 64;

    ScaledFetch<G, D, HP> fetch{p, &kv_map, items, cum, my_infos, abort_flag, l2_evict_first_policy(), smem_addr(my_ring),
                                smem_addr(my_scales), smem_addr(bars + unit * 2 * S), smem_addr(bars + unit * 2 * S + S), 0, 0, 0, lane,
                                uint32_t(31 - __clz(int(p.tokens_per_page))), 0, 0, 0, 0, 0, 0};
    uint32_t slot = 0, phase = 0;  // of the next tile to consume
    bool ok = true;

    scaled_share<G>(p, a, groups, reinterpret_cast<uint32_t*>(smem), reinterpret_cast<uint32_t*>(park_stats), share);
    uint32_t group = share->first, first_item = 0;
    while (group <= share->last) {
        const ScaledRun run = share->run(group, a.templates);
        const uint32_t run_items = run.templates;
        if (first_item >= run_items) {
            ++group;
            first_item = 0;
            continue;
        }
        const uint32_t seen = min(uint32_t(G::kItems), run_items - first_item);
        for (uint32_t i = tid; i < seen; i += G::kThreads) items[i] = scaled_item<HP>(p, a, run, first_item + i);
        __syncthreads();
        if (warp == 0) {
            const uint32_t kept = scaled_chains<false>(p, run, items, cum, seen, first_item + seen < run_items, lane);
            if (lane == 0) *pass_items = kept;
        }
        __syncthreads();
        const uint32_t count = *pass_items;
        first_item += count;
        const uint32_t tiles = cum[count];
        const uint32_t begin = uint32_t(uint64_t(tiles) * unit / U), end = uint32_t(uint64_t(tiles) * (unit + 1) / U);
        auto chain_end = [&](uint32_t chain) { return cum[chain + items[chain].length]; };

        // chains without a tile (nothing visible) publish zeros: a warp per chain
        for (uint32_t i = warp; i < count * HP; i += W) {
            const ScaledItem& it = items[i / HP];
            if (!it.active || it.chain != i / HP || chain_end(i / HP) > cum[i / HP]) continue;
            const ScaledRows rows(p, it, i % HP);
            for (uint32_t x = lane; x < uint32_t(G::kRows * (D / 4)); x += 32) {
                const uint32_t row = x / (D / 4);
                if (!rows.valid(row)) continue;
                if (p.direct != 0) scaled_publish4<T, D, true>(p, rows, &it, row, x % (D / 4) * 4, make_float4(0.0f, 0.0f, 0.0f, 0.0f));
                else if (x % (D / 4) == 0) scaled_publish_stats(p, rows, &it, row, kScaledNothing, 0.0f);
            }
        }

        ScaledState<D, NQ> st;
        uint2 q_frag[NQ][KS];
        uint32_t chain = 0xffffffffu;  // the chain the state belongs to
        bool owner = false;            // it started in this unit's share
        // state -> the chain's partial or output; of a chain held whole, or merged
        auto publish = [&]() {
            const ScaledItem* const first = items + chain;
            const ScaledRows rows(p, *first, pair);
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const uint32_t row = n * 8 + 2 * t + c;
                    if (!rows.valid(row)) continue;
                    const float sum = st.l[n][c];
                    const float up = scaled_rise(st.r[n][c], st.m[n][c]), raise = fast_exp2(up);
                    const float f = scaled_last_factor(st.r[n][c], st.m[n][c], up, sum);
                    auto part = [&](int j) {
                        return make_float4(st.acc[n][j][c] * raise * f, st.acc[n][j][2 + c] * raise * f, st.acc[n][j + 1][c] * raise * f,
                                           st.acc[n][j + 1][2 + c] * raise * f);
                    };
                    if (p.direct != 0) {
#pragma unroll
                        for (int j = 0; j < KS; j += 2) scaled_publish4<T, D, true>(p, rows, first, row, (j / 8) * 128 + g * 16 + (j % 8) * 2, part(j));
                        continue;
                    }
#pragma unroll
                    for (int j = 0; j < KS; j += 2) scaled_publish4<T, D, false>(p, rows, first, row, (j / 8) * 128 + g * 16 + (j % 8) * 2, part(j));
                    if (g == 0) scaled_publish_stats(p, rows, first, row, st.m[n][c], sum);
                }
            }
        };
        auto leave_chain = [&]() {  // the share goes on with another chain
            st.finish_sums();
            if (owner) {
                publish();
                return;
            }
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const uint32_t row = n * 8 + 2 * t + c;
                    float* dst = park + (warp * G::kRows + row) * G::kRowFloats + g * 16;
#pragma unroll
                    for (int j = 0; j < KS; j += 2) {
                        *reinterpret_cast<float4*>(dst + (j / 8) * 128 + (j % 8) * 2) =
                            make_float4(st.acc[n][j][c], st.acc[n][j][2 + c], st.acc[n][j + 1][c], st.acc[n][j + 1][2 + c]);
                    }
                    if (g == 0) {
                        park_stats[(warp * 3 + 0) * G::kRows + row] = st.m[n][c];
                        park_stats[(warp * 3 + 1) * G::kRows + row] = st.r[n][c];
                        park_stats[(warp * 3 + 2) * G::kRows + row] = st.l[n][c];
                    }
                }
            }
        };

        fetch.count = count;
        fetch.begin = begin;
        fetch.end = end;
        uint32_t next = begin;  // tile to fetch
        for (uint32_t x = begin; x < end; ++x) {
            // a pair's slot is refilled one tile later, so that its first warp rarely waits for the second
            if (pair == 0) {
                for (; ok && next < x + S - (HP - 1); ++next) ok = fetch.issue(next);
            }
            ok = ok && mbar_wait(fetch.full_bar + 8 * slot, phase, abort_flag, p);
            if (!__all_sync(0xffffffffu, ok)) {
                ok = false;
                break;
            }
            uint8_t* const codes = my_ring + slot * G::kSlotBytes;
            const uint8_t* const scales = my_scales + slot * G::kScaleBytes;
            const uint2 info = my_infos[(x - begin) & 63];
            const uint32_t tile_chain = (info.x >> 8) & 0xffu;
            if (tile_chain != chain) {
                if (chain != 0xffffffffu) leave_chain();
                chain = tile_chain;
                owner = cum[chain] >= begin;
                const ScaledRows rows(p, items[chain], pair);
                st.clear();
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    const float factor = scaled_load_q<T, D>(p, rows, n, lane, [&](int step, uint2 frag) { q_frag[n][step] = frag; });
#pragma unroll
                    for (int c = 0; c < 2; ++c) st.factor[n][c] = __shfl_sync(0xffffffffu, factor, int(8 * t + 4 * c));
                }
            }
            const uint32_t first_slot = slot;  // (moving on before the tile is 3 % faster than after it: 64 decode sequences, int8)
            if (++slot == uint32_t(S)) {
                slot = 0;
                phase ^= 1;
            }
            scaled_tile<CODE, D, NQ, HP>(p, st, codes, scales, info, items, pair, at, lane, [&](int n, int step) { return q_frag[n][step]; });
            __syncwarp();
            if (lane == 0) mbar_arrive(fetch.empty_bar + 8 * first_slot);
        }
        bool pending = false;  // the state is the start of a chain that later units' shares continue
        if (ok && chain != 0xffffffffu) {
            pending = owner && chain_end(chain) > end;
            if (pending) st.finish_sums();
            else leave_chain();
        }
        __syncthreads();
        if (*abort_flag != 0) break;
        if (pending) {
            const uint32_t last = chain_end(chain);
            for (uint32_t other_unit = unit + 1; other_unit < uint32_t(U); ++other_unit) {
                const uint32_t other_begin = uint32_t(uint64_t(tiles) * other_unit / U), other_end = uint32_t(uint64_t(tiles) * (other_unit + 1) / U);
                if (other_begin >= last) break;
                if (other_begin == other_end) continue;
                const uint32_t other = other_unit * HP + pair;
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const uint32_t row = n * 8 + 2 * t + c;
                        const float m2 = park_stats[(other * 3 + 0) * G::kRows + row], r2 = park_stats[(other * 3 + 1) * G::kRows + row];
                        const float l2 = park_stats[(other * 3 + 2) * G::kRows + row];
                        const float m1 = fmaxf(st.m[n][c], m2), r1 = fmaxf(st.r[n][c], r2);
                        st.l[n][c] = st.l[n][c] * fast_exp2(st.m[n][c] - m1) + l2 * fast_exp2(m2 - m1);
                        const float keep = fast_exp2(st.r[n][c] - r1), take = fast_exp2(r2 - r1);
                        st.m[n][c] = m1;
                        st.r[n][c] = r1;
                        const float* src = park + (other * G::kRows + row) * G::kRowFloats + g * 16;
#pragma unroll
                        for (int j = 0; j < KS; j += 2) {
                            const float4 v = *reinterpret_cast<const float4*>(src + (j / 8) * 128 + (j % 8) * 2);
                            st.acc[n][j][c] = st.acc[n][j][c] * keep + v.x * take;
                            st.acc[n][j][2 + c] = st.acc[n][j][2 + c] * keep + v.y * take;
                            st.acc[n][j + 1][c] = st.acc[n][j + 1][c] * keep + v.z * take;
                            st.acc[n][j + 1][2 + c] = st.acc[n][j + 1][2 + c] * keep + v.w * take;
                        }
                    }
                }
            }
            publish();
        }
        __syncthreads();  // items and parked states are rewritten by the next pass
    }
    scaled_drain<G>(p, fetch, pair == 0, abort_flag, lane);
}

// ------------------------------ one chain after the other, shared by all warps -------------------------------------
template <typename T, int CODE, int D, int NQ, int W>
__global__ void __launch_bounds__(W * 32, 1)
sdpa_scaled_chain_kernel(const __grid_constant__ CUtensorMap kv_map, const __grid_constant__ CUtensorMap, const MapParams p) {
    using G = ScaledGeometry<D, NQ, W, 1, false>;
    constexpr int S = G::kSlots;
    constexpr int KS = D / 16;

    extern __shared__ uint8_t smem_raw[];
    uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* const merge = reinterpret_cast<float*>(smem);  // over the ring, once a chain's copies have been consumed
    uint2* const q_frag = reinterpret_cast<uint2*>(smem + G::kBigBytes);               // [NQ][KS][32]
    float* const stat_m = reinterpret_cast<float*>(smem + G::kBigBytes + G::kQBytes);  // [W][rows]
    float* const stat_r = stat_m + W * G::kRows;
    float* const stat_l = stat_r + W * G::kRows;
    float* const row_factor = stat_l + W * G::kRows;  // [rows] from dot products to scores
    float* const row_out = row_factor + G::kRows;     // [rows] final factor of the merged accumulators
    float* const row_ref = row_out + G::kRows;        // [rows] reference of the merged accumulators
    uint8_t* const scale_ring = reinterpret_cast<uint8_t*>(stat_m) + G::kStatBytes;
    uint64_t* const bars = reinterpret_cast<uint64_t*>(scale_ring + W * S * G::kScaleBytes);
    uint2* const infos = reinterpret_cast<uint2*>(bars + W * S * 2);
    ScaledItem* const items = reinterpret_cast<ScaledItem*>(reinterpret_cast<uint8_t*>(infos) + G::kInfoBytes);
    uint32_t* const cum = reinterpret_cast<uint32_t*>(items + G::kItems);
    ScaledShare* const share = reinterpret_cast<ScaledShare*>(cum + G::kItems + 2);
    uint32_t* const pass_items = reinterpret_cast<uint32_t*>(share + 1);
    volatile uint32_t* const abort_flag = pass_items + 1;

    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t g = lane >> 2, t = lane & 3;
    if (tid == 0) {
        for (int i = 0; i < W * S; ++i) {
            mbar_init(smem_addr(bars + i / S * 2 * S + i % S), 1);
            mbar_init(smem_addr(bars + i / S * 2 * S + S + i % S), 1);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&kv_map)) : "memory");
    }
    __syncthreads();
    if constexpr (G::kSmemBytes + 14 * 1024 > 228 * 1024) {
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // (as in sdpa_map_kernel)
    }
    const ActiveCounts a = resolve_active(p);
    const uint32_t cells = p.num_kv_heads * p.head_ranges;
    const ScaledLane<D, 1> at(p.tokens_per_page, 0, lane);
    uint8_t* const my_ring = smem + warp * (S * G::kSlotBytes);
    const uint8_t* const my_scales = scale_ring + warp * (S * G::kScaleBytes);
    uint2* const my_infos = infos + warp * 64;

    ScaledFetch<G, D, 1> fetch{p, &kv_map, items, cum, my_infos, abort_flag, l2_evict_first_policy(), smem_addr(my_ring),
                               smem_addr(my_scales), smem_addr(bars + warp * 2 * S), smem_addr(bars + warp * 2 * S + S), 0, 0, 0, lane,
                               uint32_t(31 - __clz(int(p.tokens_per_page))), 0, 0, 0, 0, 0, 0};
    uint32_t slot = 0, phase = 0;
    bool ok = true;

    scaled_share<G>(p, a, cells, reinterpret_cast<uint32_t*>(smem), reinterpret_cast<uint32_t*>(stat_m), share);
    uint32_t group = share->first, first_item = 0;
    while (group <= share->last) {
        const ScaledRun run = share->run(group, a.templates);
        const uint32_t run_items = run.templates;
        if (first_item >= run_items) {
            ++group;
            first_item = 0;
            continue;
        }
        const uint32_t seen = min(uint32_t(G::kItems), run_items - first_item);
        for (uint32_t i = tid; i < seen; i += G::kThreads) items[i] = scaled_item<1>(p, a, run, first_item + i);
        __syncthreads();
        if (warp == 0) {
            const uint32_t kept = scaled_chains<true>(p, run, items, cum, seen, first_item + seen < run_items, lane);
            if (lane == 0) *pass_items = kept;
        }
        __syncthreads();
        const uint32_t count = *pass_items;
        first_item += count;
        const uint32_t tiles = cum[count];
        if (!items[0].active) {
            __syncthreads();  // the items are rewritten by the next pass
            continue;
        }
        const ScaledRows rows(p, items[0]);
        for (uint32_t n = warp; n < uint32_t(NQ); n += W) {
            const float factor = scaled_load_q<T, D>(p, rows, n, lane, [&](int step, uint2 frag) { q_frag[(n * KS + step) * 32 + lane] = frag; });
            if (t == 0) row_factor[n * 8 + g] = factor;
        }
        // the merge of the chain before wrote over the ring through ordinary stores: its copies land after them
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();

        const uint32_t begin = uint32_t(uint64_t(tiles) * warp / W), end = uint32_t(uint64_t(tiles) * (warp + 1) / W);
        ScaledState<D, NQ> st;
        st.clear();
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            st.factor[n][0] = row_factor[n * 8 + 2 * t];
            st.factor[n][1] = row_factor[n * 8 + 2 * t + 1];
        }
        fetch.count = count;
        fetch.begin = begin;
        fetch.end = end;
        uint32_t next = begin;
        for (uint32_t x = begin; x < end; ++x) {
            for (; ok && next < x + S; ++next) ok = fetch.issue(next);
            ok = ok && mbar_wait(fetch.full_bar + 8 * slot, phase, abort_flag, p);
            if (!__all_sync(0xffffffffu, ok)) {
                ok = false;
                break;
            }
            scaled_tile<CODE, D, NQ, 1>(p, st, my_ring + slot * G::kSlotBytes, my_scales + slot * G::kScaleBytes, my_infos[(x - begin) & 63],
                                        items, 0, at, lane, [&](int n, int step) { return q_frag[(n * KS + step) * 32 + lane]; });
            __syncwarp();
            if (lane == 0) mbar_arrive(fetch.empty_bar + 8 * slot);
            if (++slot == uint32_t(S)) {
                slot = 0;
                phase ^= 1;
            }
        }

        // ---- merge the warps' states and publish
        st.finish_sums();
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                if (g == 0) {
                    const uint32_t row = warp * G::kRows + n * 8 + 2 * t + c;
                    stat_m[row] = st.m[n][c];
                    stat_r[row] = st.r[n][c];
                    stat_l[row] = st.l[n][c];
                }
            }
        }
        __syncthreads();
        if (*abort_flag != 0) break;
        for (uint32_t row = tid; row < uint32_t(G::kRows); row += G::kThreads) {
            float top_m = kScaledNothing, top_r = kScaledNothing, sum = 0.0f;
            for (int w = 0; w < W; ++w) {
                top_m = fmaxf(top_m, stat_m[w * G::kRows + row]);
                top_r = fmaxf(top_r, stat_r[w * G::kRows + row]);
            }
            for (int w = 0; w < W; ++w) sum += stat_l[w * G::kRows + row] * fast_exp2(stat_m[w * G::kRows + row] - top_m);
            const float up = scaled_rise(top_r, top_m);
            row_ref[row] = top_r - up;
            row_out[row] = scaled_last_factor(top_r, top_m, up, sum);
            if (p.direct == 0 && rows.valid(row)) scaled_publish_stats(p, rows, items, row, top_m, sum);
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const float scale = fast_exp2(st.r[n][c] - row_ref[n * 8 + 2 * t + c]);
                float* dst = merge + (warp * 8 + 2 * t + c) * G::kRowFloats + g * 16;
#pragma unroll
                for (int j = 0; j < KS; j += 2) {
                    *reinterpret_cast<float4*>(dst + (j / 8) * 128 + (j % 8) * 2) =
                        make_float4(st.acc[n][j][c] * scale, st.acc[n][j][2 + c] * scale, st.acc[n][j + 1][c] * scale,
                                    st.acc[n][j + 1][2 + c] * scale);
                }
            }
            __syncthreads();
            for (uint32_t i = tid; i < 8 * D / 4; i += G::kThreads) {
                const uint32_t row = i / (D / 4), d = i % (D / 4) * 4;
                float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                for (int w = 0; w < W; ++w) {
                    const float4 v = *reinterpret_cast<const float4*>(merge + (w * 8 + row) * G::kRowFloats + d);
                    sum.x += v.x;
                    sum.y += v.y;
                    sum.z += v.z;
                    sum.w += v.w;
                }
                if (rows.valid(n * 8 + row)) {
                    const float f = row_out[n * 8 + row];
                    const float4 v = make_float4(sum.x * f, sum.y * f, sum.z * f, sum.w * f);
                    if (p.direct != 0) scaled_publish4<T, D, true>(p, rows, items, n * 8 + row, d, v);
                    else scaled_publish4<T, D, false>(p, rows, items, n * 8 + row, d, v);
                }
            }
            __syncthreads();
        }
    }
    scaled_drain<G>(p, fetch, true, abort_flag, lane);
}

}  // namespace kh
