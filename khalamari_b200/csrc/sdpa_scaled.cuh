// Map / direct attention kernel over scaled 8-bit pages (scaled_kv.cuh), for tasks of any number of Q rows.
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
// relative to. A weight is then at most 2^8 whatever the V scales are, and rounding it to f16 costs at most 2^-12 of
// the term it multiplies; one reference for both would push the weights of tokens with small V rows out of f16's
// range. The output is O * 2^(r - m) / l.
//
// Each lane copies (cp.async, 16 bytes) exactly the bytes its own MMA fragments are made of: a sum over the head
// dimension does not care about order, so lane (g, t) of the 8 x 4 lane grid takes chunks t, t + 4, .. of K rows g and
// g + 8, four consecutive codes standing in for the fragment's index pairs (2t, 2t + 1) and (2t + 8, 2t + 9), with Q
// read in the same order; and 16-byte column g of V rows 2t, 2t + 1, 2t + 8, 2t + 9, which are the fragment's tokens.
// The copies land in lane order, so that neither side of the staging buffer has a bank conflict, a swizzle or a
// transposing load, and a lane needs no barrier to read what it copied itself.
#pragma once

#include "scaled_kv.cuh"
#include "sdpa_map.cuh"

namespace kh {

// D: head dimension. NQ: n-tiles of 8 Q rows an item holds. W: warps.
template <int D, int NQ, int W>
struct ScaledGeometry {
    static_assert(D == 128 || D == 256, "head_dim 128 or 256");
    static constexpr int kThreads = W * 32;
    static constexpr int kTileTokens = 16;
    static constexpr int kRows = 8 * NQ;
    static constexpr int kChain = 64;                             // items of one pass at most
    static constexpr int kScaleOffset = 2 * kTileTokens * D;      // [K/V][16] scale bytes behind the codes
    static constexpr int kSlotBytes = kScaleOffset + 48;          // + first token and item of the tile
    static constexpr int kQBytes = NQ * (D / 16) * 32 * 8;        // Q fragments, one 8-byte pair per lane and k-step
    static constexpr int kMergeRow = D + 4;
    static constexpr int kMergeBytes = W * 8 * kMergeRow * 4;     // one n-tile of every warp
    static constexpr int kStatBytes = W * kRows * 12 + kRows * 12;
    static constexpr int kItemBytes = kChain * 48 + (kChain + 2) * 4 + 64;
    static constexpr int kFixedBytes = kQBytes + kStatBytes + kItemBytes + 256;
    static constexpr int kSmemLimit = 227 * 1024;
    static constexpr int kSlotsFit = (kSmemLimit - kFixedBytes) / (W * kSlotBytes);
    static constexpr int kSlots = kSlotsFit > 4 ? 4 : kSlotsFit;
    static constexpr int kRingBytes = W * kSlots * kSlotBytes;
    static constexpr int kBigBytes = kRingBytes > kMergeBytes ? kRingBytes : kMergeBytes;  // the merge reuses the ring
    static constexpr int kSmemBytes = kBigBytes + kFixedBytes;
    static_assert(kSlots >= 2, "staging ring too small");
    static_assert(kSmemBytes <= kSmemLimit, "shared memory");
    static_assert(kSlotBytes % 16 == 0 && kRingBytes % 16 == 0, "16-byte copies");
};

// A work item: one map task template x KV head x Q-head range x block of kRows Q rows.
struct ScaledItem {
    uint32_t tmpl, cell;        // cell = KV head x Q-head range
    uint32_t range;             // Q range index: items of equal range and cell are slices of the same rows
    uint32_t tok_begin, num_toks, row_begin;
    uint32_t kv_begin, kv_end;  // clipped to what some row of the block sees
    uint32_t all_begin, all_end; // tokens that every row of the block sees
    uint32_t req_slot;
    uint32_t active;
};
static_assert(sizeof(ScaledItem) == 48, "item size");

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_8(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// Visible range of Q token `tok` (an index into the range's tokens) cut to the item's template range.
__device__ __forceinline__ void scaled_visible(const MapParams& p, const ScaledItem& it, uint32_t tok, uint32_t kv_begin,
                                               uint32_t kv_end, uint32_t& lo, uint32_t& hi) {
    lo = kv_begin;
    hi = kv_end;
    if (p.visible != nullptr) {
        lo = max(lo, p.visible[(uint64_t(it.tok_begin) + tok) * 2]);
        hi = min(hi, p.visible[(uint64_t(it.tok_begin) + tok) * 2 + 1]);
    }
}

// Item number -> template, cell, row block, with the early-return rules of decode_task (sdpa_map.cuh).
__device__ __forceinline__ ScaledItem scaled_item(const MapParams& p, const ActiveCounts& a, uint64_t index, uint32_t rows_per_block,
                                                  uint32_t row_blocks) {
    ScaledItem it;
    it.active = 0;
    it.kv_begin = it.kv_end = it.all_begin = it.all_end = 0;
    it.tok_begin = it.num_toks = it.req_slot = 0;
    const uint32_t block = uint32_t(index % row_blocks);
    const uint64_t task = index / row_blocks;  // cell-major: the slices of one KV head's rows are neighbours
    it.tmpl = uint32_t(task % a.templates);
    it.cell = uint32_t(task / a.templates);
    it.row_begin = block * rows_per_block;
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
    if (it.row_begin >= it.num_toks * p.heads_per_task) return it;  // no Q row in this block
    it.req_slot = p.req_slots[it.tok_begin];
    if (it.req_slot >= p.num_req_slots ||
        (kv_end > kv_begin &&
         (uint64_t(kv_end) + p.tokens_per_page - 1) / p.tokens_per_page > p.pages_per_request_layer)) {
        atomicOr(p.status, kStatusMetadataOutOfRange);  // the task is dropped, as in decode_task
        return it;
    }
    it.active = 1;
    const uint32_t first = it.row_begin / p.heads_per_task;
    const uint32_t last = min((it.row_begin + rows_per_block - 1) / p.heads_per_task, it.num_toks - 1);
    uint32_t any_lo = 0xffffffffu, any_hi = 0, all_lo = 0, all_hi = 0xffffffffu;
    for (uint32_t tok = first; tok <= last; ++tok) {
        uint32_t lo, hi;
        scaled_visible(p, it, tok, kv_begin, kv_end, lo, hi);
        all_lo = max(all_lo, lo);
        all_hi = min(all_hi, hi);
        if (hi > lo) {
            any_lo = min(any_lo, lo);
            any_hi = max(any_hi, hi);
        }
    }
    if (any_hi > any_lo) {
        it.kv_begin = any_lo;
        it.kv_end = any_hi;
    }
    it.all_begin = all_lo;
    it.all_end = all_hi;
    return it;
}

// First item of CTA `cta`'s contiguous share. Costs are tiles plus a fixed term per template, prefix-summed in
// `prefix` [templates + 1]; item k of a template costs the template's cost, items are cell-major.
__device__ __forceinline__ uint64_t scaled_share(const uint32_t* prefix, uint32_t templates, uint32_t cells, uint32_t row_blocks,
                                                 uint32_t cta, uint32_t ctas) {
    const uint64_t per_cell = uint64_t(prefix[templates]) * row_blocks;
    const uint64_t total = per_cell * cells;
    const uint64_t x = total / ctas * cta + total % ctas * cta / ctas;
    const uint64_t cell = x / per_cell;
    if (cell >= cells) return uint64_t(cells) * templates * row_blocks;
    const uint64_t y = x % per_cell;
    uint32_t lo = 0, hi = templates;  // the last template that starts at or before y
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (uint64_t(prefix[mid]) * row_blocks <= y) lo = mid;
        else hi = mid;
    }
    const uint32_t cost = prefix[lo + 1] - prefix[lo];
    const uint64_t block = (y - uint64_t(prefix[lo]) * row_blocks + cost - 1) / cost;  // first item starting at or after y
    return (cell * templates + lo) * row_blocks + block;
}

template <typename T, int CODE, int D, int NQ, int W>
__global__ void __launch_bounds__(W * 32, 1)
sdpa_scaled_kernel(const __grid_constant__ CUtensorMap, const __grid_constant__ CUtensorMap, const MapParams p) {
    using G = ScaledGeometry<D, NQ, W>;
    constexpr int S = G::kSlots;
    constexpr int KC = D / 64;   // 16-byte K chunks per lane and row
    constexpr int VG = D / 128;  // 16-byte V chunks per lane and token
    constexpr int KS = D / 16;   // k-steps of Q K^T, and 16-row tiles of O^T
    constexpr float kRaise = 8.0f;
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;

    extern __shared__ __align__(16) uint8_t smem[];
    uint8_t* const ring = smem;
    float* const merge = reinterpret_cast<float*>(smem);
    uint2* const q_frag = reinterpret_cast<uint2*>(smem + G::kBigBytes);             // [NQ][KS][32]
    float* const stat_m = reinterpret_cast<float*>(smem + G::kBigBytes + G::kQBytes);  // [W][rows]
    float* const stat_r = stat_m + W * G::kRows;
    float* const stat_l = stat_r + W * G::kRows;
    float* const row_factor = stat_l + W * G::kRows;  // [rows] score scale of the row's normalised Q
    float* const row_out = row_factor + G::kRows;     // [rows] final factor of the merged accumulators
    float* const row_ref = row_out + G::kRows;        // [rows] merged value reference
    ScaledItem* const items = reinterpret_cast<ScaledItem*>(row_ref + G::kRows);
    uint32_t* const cum = reinterpret_cast<uint32_t*>(items + G::kChain);  // [kChain + 1] first tile of every item
    uint32_t* const pass = cum + G::kChain + 2;                            // [0] items of this pass; scan scratch

    const uint32_t tid = threadIdx.x;
    const uint32_t warp = tid >> 5, lane = tid & 31;
    const uint32_t g = lane >> 2, t = lane & 3;
    const uint32_t P = p.tokens_per_page;

    if constexpr (G::kSmemBytes + 14 * 1024 > 228 * 1024) {
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // (as in sdpa_map_kernel)
    }
    const ActiveCounts a = resolve_active(p);
    const uint32_t cells = p.num_kv_heads * p.head_ranges;
    const uint32_t rows_per_task = p.max_q_tokens * p.heads_per_task;
    const uint32_t row_blocks = (rows_per_task + G::kRows - 1) / G::kRows;
    const uint64_t total_items = uint64_t(a.templates) * cells * row_blocks;

    // ---- this CTA's items [item, item_end)
    uint64_t item, item_end;
    if (total_items <= gridDim.x) {
        item = min(uint64_t(blockIdx.x), total_items);
        item_end = min(item + 1, total_items);
    } else if (a.templates <= kBalanceMaxTemplates && (a.templates + 1) * 4 <= uint32_t(G::kBigBytes)) {
        // prefix sum of the templates' costs, in the ring (nothing has been copied yet)
        uint32_t* const prefix = reinterpret_cast<uint32_t*>(ring);
        const uint32_t chunk = (a.templates + G::kThreads - 1) / G::kThreads;
        const uint32_t first = min(tid * chunk, a.templates), last = min(first + chunk, a.templates);
        for (uint32_t i = tid; i < a.templates; i += G::kThreads) {
            const uint32_t q_range = p.templates[uint64_t(i) * 3];
            const uint32_t b = p.templates[uint64_t(i) * 3 + 1], e = p.templates[uint64_t(i) * 3 + 2];
            prefix[i + 1] = (q_range == 0xffffffffu || e <= b) ? 1u : (e - b) / 16 + 3u;
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
        if (lane == 31) stat_m[warp] = __uint_as_float(scan);
        __syncthreads();
        uint32_t before = scan - sum;
        for (uint32_t w = 0; w < warp; ++w) before += __float_as_uint(stat_m[w]);
        for (uint32_t i = first; i < last; ++i) {
            before += prefix[i + 1];
            prefix[i + 1] = before;
        }
        if (tid == 0) prefix[0] = 0;
        __syncthreads();
        item = scaled_share(prefix, a.templates, cells, row_blocks, blockIdx.x, gridDim.x);
        item_end = scaled_share(prefix, a.templates, cells, row_blocks, blockIdx.x + 1, gridDim.x);
        __syncthreads();
    } else {
        item = total_items / gridDim.x * blockIdx.x + min(total_items % gridDim.x, uint64_t(blockIdx.x));
        item_end = item + total_items / gridDim.x + (blockIdx.x < total_items % gridDim.x ? 1 : 0);
    }

    const uint64_t code_bytes = uint64_t(2) * p.num_kv_heads * P * D;  // of a page
    const uint64_t plane_bytes = uint64_t(p.num_kv_heads) * P * D;
    const uint32_t ring_addr = smem_addr(ring) + warp * (S * G::kSlotBytes);
    uint8_t* const my_ring = ring + warp * (S * G::kSlotBytes);

    while (item < item_end) {
        // ---- one pass: the items of one chain - slices of the same Q rows - or a single item
        const uint32_t ahead = uint32_t(min(uint64_t(G::kChain), item_end - item));
        if (tid < ahead) items[tid] = scaled_item(p, a, item + tid, G::kRows, row_blocks);
        __syncthreads();
        if (warp == 0) {
            uint32_t length = 1;  // items of the chain
            if (row_blocks == 1 && p.direct == 0 && items[0].active) {
                for (; length < ahead; ++length) {
                    const ScaledItem& next = items[length];
                    if (!next.active || next.range != items[0].range || next.cell != items[0].cell) break;
                }
            }
            uint32_t run = 0;
            for (uint32_t base = 0; base < length; base += 32) {
                const uint32_t i = base + lane;
                uint32_t tiles = 0;
                if (i < length && items[i].kv_end > items[i].kv_begin) {
                    tiles = (items[i].kv_end + 15) / 16 - items[i].kv_begin / 16;
                }
                uint32_t scan = tiles;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const uint32_t v = __shfl_up_sync(0xffffffffu, scan, d);
                    if (lane >= uint32_t(d)) scan += v;
                }
                if (i < length) cum[i] = run + scan - tiles;
                run += __shfl_sync(0xffffffffu, scan, 31);
            }
            if (lane == 0) {
                cum[length] = run;
                pass[0] = length;
            }
        }
        __syncthreads();
        const uint32_t length = pass[0];
        const uint32_t tiles = cum[length];
        const ScaledItem head = items[0];
        item += length;
        if (!head.active) {
            __syncthreads();  // the items are rewritten by the next pass
            continue;
        }
        const uint32_t head_begin = (head.cell / p.head_ranges) * p.group + (head.cell % p.head_ranges) * p.heads_per_task;
        const uint32_t num_heads = min(p.heads_per_task, p.group - (head.cell % p.head_ranges) * p.heads_per_task);
        const uint32_t kv_head = head.cell / p.head_ranges;
        auto row_valid = [&](uint32_t row) {  // row of the block -> is it a Q row
            const uint32_t r = head.row_begin + row;
            return r / p.heads_per_task < head.num_toks && r % p.heads_per_task < num_heads;
        };

        // ---- Q fragments: warp n stages n-tile n. Lane (g, t) holds row g's elements 64 c + 16 t + (0 .. 15). bf16 rows
        // are scaled by a power of two so that their largest element lies in [2^8, 2^9): exact in f16 down to 2^-22 of
        // that element, and no bf16 value overflows.
        for (uint32_t n = warp; n < uint32_t(NQ); n += W) {
            const uint32_t row = n * 8 + g;
            uint4 raw[KC][2];
            if (row_valid(row)) {
                const uint32_t r = head.row_begin + row;
                const uint64_t q_row = (uint64_t(head.tok_begin) + r / p.heads_per_task) * p.num_q_heads + head_begin + r % p.heads_per_task;
                const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + q_row * D);
#pragma unroll
                for (int c = 0; c < KC; ++c) {
                    raw[c][0] = src[c * 8 + t * 2];
                    raw[c][1] = src[c * 8 + t * 2 + 1];
                }
            } else {
#pragma unroll
                for (int c = 0; c < KC; ++c) raw[c][0] = raw[c][1] = make_uint4(0, 0, 0, 0);
            }
            float factor = p.scale_log2e;
            float up = 1.0f;
            if constexpr (kBf16) {
                uint32_t most = 0;
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
                const int exponent = int(max(most & 0xffffu, most >> 16) >> 7);  // of the largest element, biased
                if (exponent >= 9 && exponent < 255) {  // (tinier rows and rows with a NaN or an infinity go as they are)
                    // 2^(8 - k) and 2^(k - 8), k = exponent - 127: both normal f32 values
                    up = __uint_as_float(uint32_t(min(max(262 - exponent, 1), 254)) << 23);
                    factor = p.scale_log2e * __uint_as_float(uint32_t(min(max(exponent - 8, 1), 254)) << 23);
                }
            }
            if (t == 0) row_factor[row] = factor;
#pragma unroll
            for (int c = 0; c < KC; ++c) {
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint4 v = raw[c][w / 2];
                    uint2 pair = w % 2 == 0 ? make_uint2(v.x, v.y) : make_uint2(v.z, v.w);
                    if constexpr (kBf16) {
                        const float2 x = unpack2<__nv_bfloat16>(pair.x), y = unpack2<__nv_bfloat16>(pair.y);
                        pair = make_uint2(pack2<__half>(x.x * up, x.y * up), pack2<__half>(y.x * up, y.y * up));
                    }
                    q_frag[(n * KS + c * 4 + w) * 32 + lane] = pair;
                }
            }
        }
        __syncthreads();

        // ---- this warp's tiles [begin, end) of the chain
        const uint32_t begin = uint32_t(uint64_t(tiles) * warp / W), end = uint32_t(uint64_t(tiles) * (warp + 1) / W);
        float acc[NQ][KS][4];
        float m[NQ][2], r[NQ][2], l[NQ][2], factor[NQ][2];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
#pragma unroll
            for (int j = 0; j < KS; ++j) acc[n][j][0] = acc[n][j][1] = acc[n][j][2] = acc[n][j][3] = 0.0f;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                m[n][c] = r[n][c] = -INFINITY;
                l[n][c] = 0.0f;
                factor[n][c] = row_factor[n * 8 + 2 * t + c];
            }
        }
        const uint64_t table = (uint64_t(head.req_slot) * p.num_gqa_layers + p.layer_index) * p.pages_per_request_layer;
        // Lane i of the window holds tile window_base + i: its item, first token and the pages of its two 8-token halves.
        uint32_t win_item = 0, win_tok = 0, win_page0 = 0, win_page1 = 0;
        auto load_window = [&](uint32_t base) {
            const uint32_t x = base + lane;
            win_page0 = win_page1 = 0xffffffffu;
            if (x < end) {
                uint32_t lo = 0, hi = length;
                while (hi - lo > 1) {
                    const uint32_t mid = (lo + hi) / 2;
                    if (cum[mid] <= x) lo = mid;
                    else hi = mid;
                }
                win_item = lo;
                const uint32_t kv_begin = items[lo].kv_begin, kv_end = items[lo].kv_end;
                win_tok = (kv_begin / 16 + x - cum[lo]) * 16;
                // only halves that hold a token of the item are fetched: the others' pages may not exist
                if (win_tok + 8 > kv_begin) win_page0 = p.page_ids[table + win_tok / P];
                if (win_tok + 8 < kv_end) win_page1 = p.page_ids[table + (win_tok + 8) / P];
                if ((win_tok + 8 > kv_begin && win_page0 >= p.pool_pages) || (win_tok + 8 < kv_end && win_page1 >= p.pool_pages)) {
                    atomicOr(p.status, kStatusPageOutOfPool);
                }
                if (win_page0 >= p.pool_pages) win_page0 = 0xffffffffu;
                if (win_page1 >= p.pool_pages) win_page1 = 0xffffffffu;
            }
        };
        auto issue = [&](uint32_t x) {
            if (x < end) {
                if (((x - begin) & 31) == 0) load_window(x);
                const int source = int((x - begin) & 31);
                const uint32_t it = __shfl_sync(0xffffffffu, win_item, source), tok = __shfl_sync(0xffffffffu, win_tok, source);
                uint32_t page[2] = {__shfl_sync(0xffffffffu, win_page0, source), __shfl_sync(0xffffffffu, win_page1, source)};
                const uint32_t slot = ((x - begin) % S) * G::kSlotBytes;
                const uint32_t dst = ring_addr + slot + lane * 16;
                const uint8_t* base[2];
                uint32_t bytes[2], in_page[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    bytes[h] = page[h] == 0xffffffffu ? 0u : 16u;  // nothing fetched, zeros written
                    in_page[h] = (tok + 8 * h) % P;
                    base[h] = p.kv_pages + uint64_t(bytes[h] ? page[h] : 0) * p.page_bytes;
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint8_t* k = base[h] + (uint64_t(kv_head) * P + in_page[h] + g) * D + t * 16;
#pragma unroll
                    for (int c = 0; c < KC; ++c) cp_async_16(dst + (h * KC + c) * 512, k + c * 64, bytes[h]);
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint8_t* v = base[h] + plane_bytes + (uint64_t(kv_head) * P + in_page[h] + 2 * t) * D + g * 16;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
#pragma unroll
                        for (int c = 0; c < VG; ++c) {
                            cp_async_16(dst + (2 * KC + (h * 2 + i) * VG + c) * 512, v + i * D + c * 128, bytes[h]);
                        }
                    }
                }
                if (lane < 4) {  // scale bytes: [plane][half] groups of 8
                    const uint32_t plane = lane >> 1, h = lane & 1;
                    const uint8_t* src = (h ? base[1] : base[0]) + code_bytes + (uint64_t(kv_head) * 2 + plane) * P + (h ? in_page[1] : in_page[0]);
                    cp_async_8(ring_addr + slot + G::kScaleOffset + lane * 8, src, (h ? bytes[1] : bytes[0]) / 2);
                }
                if (lane == 4) {
                    uint32_t* info = reinterpret_cast<uint32_t*>(my_ring + slot + G::kScaleOffset + 32);
                    info[0] = it;
                    info[1] = tok;
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int s = 0; s < S - 1; ++s) issue(begin + s);
        for (uint32_t x = begin; x < end; ++x) {
            issue(x + S - 1);
            asm volatile("cp.async.wait_group %0;" ::"n"(S - 1) : "memory");
            __syncwarp();  // the scale bytes and the tile's numbers came through other lanes
            uint8_t* const slot = my_ring + ((x - begin) % S) * G::kSlotBytes;
            uint4* const mine = reinterpret_cast<uint4*>(slot) + lane;
            const uint32_t it = *reinterpret_cast<const uint32_t*>(slot + G::kScaleOffset + 32);
            const uint32_t tok = *reinterpret_cast<const uint32_t*>(slot + G::kScaleOffset + 36);
            const uint8_t* const scales = slot + G::kScaleOffset;
            const float k_scale[2] = {scale_of_byte(scales[g]), scale_of_byte(scales[8 + g])};
            const float v_log[2] = {float(int(scales[16 + g]) - 127), float(int(scales[24 + g]) - 127)};

            // ---- S^T = K Q^T
            float s[NQ][4];
#pragma unroll
            for (int n = 0; n < NQ; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                const uint4 k0 = mine[c * 32], k1 = mine[(KC + c) * 32];
                const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t frag[4];
                    codes4_to_half<CODE>(w0[w], frag[0], frag[2]);
                    codes4_to_half<CODE>(w1[w], frag[1], frag[3]);
#pragma unroll
                    for (int n = 0; n < NQ; ++n) {
                        const uint2 q = q_frag[(n * KS + c * 4 + w) * 32 + lane];
                        mma_16816<__half>(s[n], frag, q.x, q.y);
                    }
                }
            }
            // ---- scores: lane (g, t) holds tokens g, g + 8 (s[0..1], s[2..3]) of rows 2t, 2t + 1. Log2 domain.
            float y[NQ][4];
            const ScaledItem& cur = items[it];
            const bool inside = tok >= cur.all_begin && tok + 16 <= cur.all_end;
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][e] *= k_scale[e / 2] * factor[n][e % 2];
            }
            if (!inside) {
                const uint32_t tmpl_begin = p.templates[uint64_t(cur.tmpl) * 3 + 1], tmpl_end = p.templates[uint64_t(cur.tmpl) * 3 + 2];
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const uint32_t row = n * 8 + 2 * t + c;
                        uint32_t lo = 0, hi = 0;
                        if (row_valid(row)) {
                            scaled_visible(p, cur, (head.row_begin + row) / p.heads_per_task, tmpl_begin, tmpl_end, lo, hi);
                        }
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t token = tok + 8 * h + g;
                            if (token < lo || token >= hi) s[n][2 * h + c] = -INFINITY;
                        }
                    }
                }
                if constexpr (CODE == kCodeE4M3) {
                    // rows past the item's end may hold anything, the NaN code among it, and 0 * NaN is NaN
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (tok + (i / 2) * 8 + 2 * t + i % 2 >= cur.kv_end) {
#pragma unroll
                            for (int c = 0; c < VG; ++c) mine[(2 * KC + i * VG + c) * 32] = make_uint4(0, 0, 0, 0);
                        }
                    }
                }
            }
            bool raise = false;
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
#pragma unroll
                for (int e = 0; e < 4; ++e) y[n][e] = s[n][e] + v_log[e / 2];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    raise = raise || fmaxf(s[n][c], s[n][2 + c]) > m[n][c] + kRaise || fmaxf(y[n][c], y[n][2 + c]) > r[n][c] + kRaise;
                }
            }
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float top_s = fmaxf(s[n][c], s[n][2 + c]), top_y = fmaxf(y[n][c], y[n][2 + c]);
#pragma unroll
                        for (int d = 4; d <= 16; d <<= 1) {
                            top_s = fmaxf(top_s, __shfl_xor_sync(0xffffffffu, top_s, d));
                            top_y = fmaxf(top_y, __shfl_xor_sync(0xffffffffu, top_y, d));
                        }
                        if (top_s > m[n][c]) {
                            l[n][c] *= fast_exp2(m[n][c] - top_s);  // (0 from -inf)
                            m[n][c] = top_s;
                        }
                        if (top_y > r[n][c]) {
                            const float keep = fast_exp2(r[n][c] - top_y);
                            r[n][c] = top_y;
#pragma unroll
                            for (int j = 0; j < KS; ++j) {
                                acc[n][j][c] *= keep;
                                acc[n][j][2 + c] *= keep;
                            }
                        }
                    }
                }
            }
            // ---- probabilities into the sum, value weights as B fragments (packed pairs of rows, transposed)
            uint32_t weight[NQ][2];
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                float w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float ms = m[n][e % 2] == -INFINITY ? 0.0f : m[n][e % 2], rs = r[n][e % 2] == -INFINITY ? 0.0f : r[n][e % 2];
                    l[n][e % 2] += fast_exp2(s[n][e] - ms);
                    w[e] = fast_exp2(y[n][e] - rs);
                }
                weight[n][0] = movmatrix_trans(pack2<__half>(w[0], w[1]));
                weight[n][1] = movmatrix_trans(pack2<__half>(w[2], w[3]));
            }
            // ---- O^T += V^T P^T: lane (g, t) has codes 16 g .. of tokens 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
            for (int c = 0; c < VG; ++c) {
                uint4 v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = mine[(2 * KC + i * VG + c) * 32];
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint32_t v0 = w == 0 ? v[0].x : w == 1 ? v[0].y : w == 2 ? v[0].z : v[0].w;
                    const uint32_t v1 = w == 0 ? v[1].x : w == 1 ? v[1].y : w == 2 ? v[1].z : v[1].w;
                    const uint32_t v2 = w == 0 ? v[2].x : w == 1 ? v[2].y : w == 2 ? v[2].z : v[2].w;
                    const uint32_t v3 = w == 0 ? v[3].x : w == 1 ? v[3].y : w == 2 ? v[3].z : v[3].w;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        // bytes 2j, 2j + 1 of the four tokens: [token pair][byte]
                        uint32_t frag[4];
                        codes4_to_half<CODE>(__byte_perm(v0, v1, j == 0 ? 0x5140 : 0x7362), frag[0], frag[1]);
                        codes4_to_half<CODE>(__byte_perm(v2, v3, j == 0 ? 0x5140 : 0x7362), frag[2], frag[3]);
#pragma unroll
                        for (int n = 0; n < NQ; ++n) mma_16816<__half>(acc[n][c * 8 + w * 2 + j], frag, weight[n][0], weight[n][1]);
                    }
                }
            }
            __syncwarp();  // the slot's scale bytes have been read by every lane before another copy lands in it
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");

        // ---- merge the warps' states and publish
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int d = 4; d <= 16; d <<= 1) l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], d);
                if (g == 0) {
                    const uint32_t row = warp * G::kRows + n * 8 + 2 * t + c;
                    stat_m[row] = m[n][c];
                    stat_r[row] = r[n][c];
                    stat_l[row] = l[n][c];
                }
            }
        }
        __syncthreads();
        for (uint32_t row = tid; row < uint32_t(G::kRows); row += G::kThreads) {
            float top_m = -INFINITY, top_r = -INFINITY, sum = 0.0f;
            for (int w = 0; w < W; ++w) {
                top_m = fmaxf(top_m, stat_m[w * G::kRows + row]);
                top_r = fmaxf(top_r, stat_r[w * G::kRows + row]);
            }
            for (int w = 0; w < W; ++w) {
                const float mw = stat_m[w * G::kRows + row];
                sum += stat_l[w * G::kRows + row] * (mw == -INFINITY ? 0.0f : fast_exp2(mw - top_m));
            }
            row_ref[row] = top_r;
            row_out[row] = sum == 0.0f ? 0.0f : fast_exp2(top_r - top_m) / sum;  // (a NaN sum stays NaN)
            if (p.direct == 0 && row_valid(row)) {
                const uint32_t rr = head.row_begin + row;
                const uint64_t index = (uint64_t(head.tmpl) * p.num_q_heads + head_begin + rr % p.heads_per_task) * p.max_q_tokens + rr / p.heads_per_task;
                p.partial_sum[index] = sum;
                // natural-log domain; a NaN sum needs a finite maximum to reach the merged output
                p.partial_max[index] = top_m > -INFINITY ? top_m * 0.6931471805599453f : (sum == sum ? -INFINITY : 0.0f);
                // the chain's other slices publish empty partials
                for (uint32_t i = 1; i < length; ++i) {
                    const uint64_t other = index + uint64_t(items[i].tmpl - head.tmpl) * p.num_q_heads * p.max_q_tokens;
                    p.partial_sum[other] = 0.0f;
                    p.partial_max[other] = -INFINITY;
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const float top_r = row_ref[n * 8 + 2 * t + c];
                const float scale = r[n][c] == -INFINITY ? 0.0f : fast_exp2(r[n][c] - top_r);
                float* dst = merge + (warp * 8 + 2 * t + c) * G::kMergeRow + g * 16;
#pragma unroll
                for (int j = 0; j < KS; j += 2) {
                    *reinterpret_cast<float4*>(dst + (j / 8) * 128 + (j % 8) * 2) =
                        make_float4(acc[n][j][c] * scale, acc[n][j][2 + c] * scale, acc[n][j + 1][c] * scale, acc[n][j + 1][2 + c] * scale);
                }
            }
            __syncthreads();
            for (uint32_t i = tid; i < 8 * D / 4; i += G::kThreads) {
                const uint32_t row = i / (D / 4), d = i % (D / 4) * 4;
                float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                for (int w = 0; w < W; ++w) {
                    const float4 v = *reinterpret_cast<const float4*>(merge + (w * 8 + row) * G::kMergeRow + d);
                    sum.x += v.x;
                    sum.y += v.y;
                    sum.z += v.z;
                    sum.w += v.w;
                }
                if (row_valid(n * 8 + row)) {
                    const float f = row_out[n * 8 + row];
                    const float4 v = make_float4(sum.x * f, sum.y * f, sum.z * f, sum.w * f);
                    const uint32_t rr = head.row_begin + n * 8 + row;
                    const uint32_t q_head = head_begin + rr % p.heads_per_task, tok = rr / p.heads_per_task;
                    if (p.direct != 0) {
                        store_out4<T>(static_cast<T*>(p.out) + ((uint64_t(head.tok_begin) + tok) * p.num_q_heads + q_head) * D + d, v);
                    } else {
                        const uint64_t index = (uint64_t(head.tmpl) * p.num_q_heads + q_head) * p.max_q_tokens + tok;
                        *reinterpret_cast<float4*>(p.partial_out + index * D + d) = v;
                    }
                }
            }
            __syncthreads();
        }
    }
}

}  // namespace kh
