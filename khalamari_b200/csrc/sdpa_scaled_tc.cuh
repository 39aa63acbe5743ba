// Attention over scaled 8-bit pages (scaled_kv.cuh) for wide Q tiles (prefill, up to 128 rows a task) at head_dim 128, on
// the 5th-generation tensor cores.
//
//   S = Q K^T    tcgen05.mma kind::f16, M = 128 rows, N = 128 tokens; Q and K in shared memory, S in tensor memory.
//   O += P V     P from tensor memory (over the columns of the S it came from), V in shared memory, O in tensor memory.
//
// Codes become 16-bit operands of the Q/output type once per step of 128 tokens, in shared memory, with their row's
// power-of-two scale already applied: int8 and E4M3 codes times 2^e are exact in bf16, and in f16 as far as its range goes
// (results are rounded below 2^-14 and saturate at 65504, as values of an f16 cache would). Two Q tiles of the same
// sequence and KV head share every converted step and take turns: while the softmax of one tile runs, the tensor cores
// work on the other's products.
//
// What bounds it: an exponential for every score (16 a cycle and SM: 1,024 cycles for a tile's 128 x 128 scores, which is
// also about what its two products take), then instruction issue, of which the conversion takes about a third - hence
// the two tiles per conversion.
//
// Warps: 0-3 softmax and epilogue of tile A (one thread a row), 4-7 of tile B, 8-13 conversion, 14 task decoding and
// copies, 15 tensor-core issue (one thread). All waits are bounded (mbar_wait); no named barriers between roles.
#pragma once

#include "scaled_kv.cuh"
#include "sdpa_map.cuh"
#include "sdpa_scaled.cuh"
#include "sdpa_tc.cuh"

namespace kh {

struct ScaledTc {
    static constexpr int kD = 128;
    static constexpr int kRows = 128;
    static constexpr int kStep = 128;                            // tokens of a step
    static constexpr int kChunks = kStep / 16;                   // raw slots (16 tokens) of a step
    static constexpr int kRawSlots = 8;
    static constexpr int kRawBytes = 2 * 16 * kD;
    static constexpr int kOperandBytes = kStep * kD * 2;         // a step's K or V, and a Q tile: two 64-element halves of
    static constexpr int kHalfBytes = kOperandBytes / 2;         // [128 rows][128 bytes], 128-byte swizzle
    static constexpr int kConverters = 6;
    static constexpr int kThreads = 16 * 32;
    static constexpr int kSmemBytes = 6 * kOperandBytes + kRawSlots * (kRawBytes + 32) + 1024 + 1024;
    static_assert(kSmemBytes <= 227 * 1024, "shared memory");
};

// Two Q tiles (or one: B inactive) over one KV range of one request and KV head.
struct ScaledTcTask {
    uint32_t done, active_b;
    uint32_t req_slot, kv_head;
    uint32_t begin, end;       // what some row of the tiles sees
    uint32_t first;            // begin, rounded down to a multiple of 16
    uint32_t steps;
    uint32_t tmpl[2], head_begin, num_heads;
    uint32_t tok_begin[2], num_toks[2], kv_begin[2], kv_end[2];
};

// 2^(b - 127) as packed pairs of T, in two factors: f16 scales may lie below its smallest normal number, and the product
// of a code with the first factor is exact. Where V's byte marks a row that is not finite its codes count as zeros (the
// row's K is NaN, which is what reaches the queries that see it).
template <typename T>
__device__ __forceinline__ void scaled_factors(uint32_t b, bool v, uint32_t& first, uint32_t& second);
template <>
__device__ __forceinline__ void scaled_factors<__nv_bfloat16>(uint32_t b, bool v, uint32_t& first, uint32_t& second) {
    if (v && b == 255) b = 0;
    first = (b << 7) * 0x00010001u;
    second = 0;
}
template <>
__device__ __forceinline__ void scaled_factors<__half>(uint32_t b, bool v, uint32_t& first, uint32_t& second) {
    if (b == 255 || b == 0) {
        first = b == 0 || v ? 0u : 0x7c007c00u;
        second = 0x3c003c00u;
        return;
    }
    const int e = int(b) - 127;
    const int high = max(min(e, 15), -14), rest = max(min(e - high, 15), -24);
    first = uint32_t((high + 15) << 10) * 0x00010001u;
    // (below 2^-14 a subnormal power; scales below 2^-38 leave nothing of a code either way)
    second = (rest >= -14 ? uint32_t((rest + 15) << 10) : 1u << (rest + 24)) * 0x00010001u;
}

template <typename T>
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b);
template <>
__device__ __forceinline__ uint32_t mul2<__nv_bfloat16>(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <>
__device__ __forceinline__ uint32_t mul2<__half>(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// Four codes to four elements of T, exactly, unscaled.
template <typename T, int CODE>
__device__ __forceinline__ void codes4_to(uint32_t word, uint32_t& lo, uint32_t& hi) {
    if constexpr (std::is_same<T, __half>::value) {
        codes4_to_half<CODE>(word, lo, hi);
    } else if constexpr (CODE == kCodeInt8) {
        // bf16 has 8 significant bits: 128 + (c & 127) minus 128 (c >= 0) or 256 (c < 0), whose patterns are 0x4300 with
        // the code's low seven bits and 0x4300 with its sign bit
        const uint32_t a = __byte_perm(word, 0x43434343u, 0x4140), b = __byte_perm(word, 0x43434343u, 0x4342);
        asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(lo) : "r"(a & 0xff7fff7fu), "r"(a & 0xff80ff80u));
        asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(hi) : "r"(b & 0xff7fff7fu), "r"(b & 0xff80ff80u));
    } else {
        lo = fp8x2_high_bytes_to_t2<__nv_bfloat16>(__byte_perm(word, 0u, 0x1404));
        hi = fp8x2_high_bytes_to_t2<__nv_bfloat16>(__byte_perm(word, 0u, 0x3424));
    }
}

// A wait of a whole warp: the same answer in every lane.
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag, const MapParams& p) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, p));
}

template <typename T, int CODE>
__global__ void __launch_bounds__(ScaledTc::kThreads, 1)
sdpa_scaled_tc_kernel(const __grid_constant__ CUtensorMap kv_map, const __grid_constant__ CUtensorMap, const MapParams p) {
    using G = ScaledTc;
    constexpr int D = G::kD;
    constexpr float kRescaleLog2 = 8.0f;  // O is rescaled only when a row maximum grows by more than 2^8
    // bf16 probabilities carry their rounding remainder in a second product where it counts; f16 ones (11 bits) do not
    constexpr bool kRemainder = std::is_same<T, __nv_bfloat16>::value;

    extern __shared__ uint8_t smem_raw[];
    uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* const q_tile = smem;                                  // [2]
    uint8_t* const k_ring = smem + 2 * G::kOperandBytes;           // [2]
    uint8_t* const v_ring = smem + 4 * G::kOperandBytes;           // [2]
    uint8_t* const raw_ring = smem + 6 * G::kOperandBytes;         // [kRawSlots]
    uint8_t* const raw_scales = raw_ring + G::kRawSlots * G::kRawBytes;
    ScaledTcTask* const tasks = reinterpret_cast<ScaledTcTask*>(raw_scales + G::kRawSlots * 32);  // [2]
    uint64_t* const bars = reinterpret_cast<uint64_t*>(tasks + 2);
    const uint32_t bar0 = smem_addr(bars);
    const uint32_t raw_full = bar0, raw_empty = bar0 + 64;         // [8] each
    const uint32_t k_full = bar0 + 128, k_empty = bar0 + 144, v_full = bar0 + 160, v_empty = bar0 + 176;  // [2] each
    const uint32_t s_full = bar0 + 192, p_full = bar0 + 208, q_full = bar0 + 224;  // [tile]
    const uint32_t o_full = bar0 + 240, o_free = bar0 + 256, pv_done = bar0 + 272;
    const uint32_t task_full = bar0 + 288, task_empty = bar0 + 304;  // [2]
    const uint32_t drain = bar0 + 320;
    constexpr int kBars = 41;
    volatile uint32_t* const abort_flag = reinterpret_cast<volatile uint32_t*>(bars + kBars);
    uint32_t* const tmem_slot = const_cast<uint32_t*>(abort_flag) + 1;
    volatile uint32_t* const remainder_flag = abort_flag + 2;      // [2][4]
    static_assert(sizeof(ScaledTcTask) * 2 + kBars * 8 + 48 <= 1024, "small shared memory");

    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < G::kRawSlots; ++i) {
            mbar_init(raw_full + 8 * i, 1);
            mbar_init(raw_empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(k_full + 8 * i, G::kChunks);
            mbar_init(v_full + 8 * i, G::kChunks);
            mbar_init(k_empty + 8 * i, 1);
            mbar_init(v_empty + 8 * i, 1);
            mbar_init(s_full + 8 * i, 1);
            mbar_init(p_full + 8 * i, 4);
            mbar_init(q_full + 8 * i, 4);
            mbar_init(o_full + 8 * i, 1);
            mbar_init(o_free + 8 * i, 4);
            mbar_init(pv_done + 8 * i, 1);
            mbar_init(task_full + 8 * i, 1);
            mbar_init(task_empty + 8 * i, 8 + G::kConverters + 1);
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint32_t tmem_s = tmem, tmem_o = tmem + 256;             // + 128 * tile; P over the first 64 columns of S
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const ActiveCounts a = resolve_active(p);

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == 14) {
            // ------------------------------ tasks and copies --------------------------------------------------------
            // Tasks are pairs of neighbouring templates, dealt round robin KV head by KV head, so that at any moment the
            // CTAs read the same K/V rows through L2; within a head from the last template to the first, so that the
            // long rows of a causal batch do not come last.
            const uint32_t cells = p.num_kv_heads * p.head_ranges;
            // (few tasks: one tile each, on as many SMs)
            const uint32_t stride = uint64_t(a.templates) * cells >= 2 * uint64_t(gridDim.x) ? 2 : 1;
            const uint32_t pairs = (a.templates + stride - 1) / stride;
            const uint64_t total = uint64_t(pairs) * cells;
            const uint32_t page_shift = 31 - __clz(int(p.tokens_per_page));
            const uint64_t policy = l2_evict_first_policy();
            uint32_t published = 0, issued = 0;
            bool ok = true;
            auto decode = [&](uint32_t tmpl, uint32_t tile, ScaledTcTask& task) -> bool {
                if (tmpl >= a.templates) return false;
                const uint32_t range = p.templates[uint64_t(tmpl) * 3];
                uint32_t begin, end;
                if (p.q_ranges == nullptr) {
                    if (range >= a.tokens) return false;
                    begin = range;
                    end = range + 1;
                } else {
                    if (range >= a.q_tiles) return false;
                    begin = p.q_ranges[range * 2];
                    end = p.q_ranges[range * 2 + 1];
                    if (begin >= a.tokens || end > a.tokens || end <= begin) return false;
                }
                const uint32_t kv_begin = p.templates[uint64_t(tmpl) * 3 + 1], kv_end = p.templates[uint64_t(tmpl) * 3 + 2];
                const uint32_t slot = p.req_slots[begin];
                if (slot >= p.num_req_slots ||
                    (kv_end > kv_begin && (uint64_t(kv_end) + p.tokens_per_page - 1) / p.tokens_per_page > p.pages_per_request_layer)) {
                    if (lane == 0) atomicOr(p.status, kStatusMetadataOutOfRange);
                    return false;
                }
                task.tmpl[tile] = tmpl;
                task.tok_begin[tile] = begin;
                task.num_toks[tile] = min(end - begin, p.max_q_tokens);
                // what some row of the tile sees
                uint32_t lo = 0xffffffffu, hi = 0;
                for (uint32_t tok = lane; tok < task.num_toks[tile]; tok += 32) {
                    uint32_t l, h;
                    scaled_visible(p, begin, tok, kv_begin, kv_end, l, h);
                    if (h > l) {
                        lo = min(lo, l);
                        hi = max(hi, h);
                    }
                }
                lo = __reduce_min_sync(0xffffffffu, lo);
                hi = __reduce_max_sync(0xffffffffu, hi);
                task.kv_begin[tile] = hi > lo ? lo : 0;
                task.kv_end[tile] = hi > lo ? hi : 0;
                if (tile == 0) task.req_slot = slot;
                return tile == 0 || slot == task.req_slot;
            };
            // publishes the task and streams its raw slots
            auto stream = [&](ScaledTcTask& task) {
                if (!ok) return;
                task.begin = task.kv_begin[0];
                task.end = task.kv_end[0];
                if (task.active_b) task.end = max(task.end, task.kv_end[1]);  // (tiles together begin together)
                task.first = task.begin / 16 * 16;
                task.steps = task.end > task.first ? (task.end - task.first + G::kStep - 1) / G::kStep : 0;
                const uint32_t ts = published & 1;
                if (!mbar_wait_warp(task_empty + 8 * ts, ((published >> 1) & 1) ^ 1, abort_flag, p)) {
                    ok = false;
                    return;
                }
                if (lane == 0) {
                    tasks[ts] = task;
                    mbar_arrive(task_full + 8 * ts);
                }
                ++published;
                if (task.done) return;
                const uint64_t table = (uint64_t(task.req_slot) * p.num_gqa_layers + p.layer_index) * p.pages_per_request_layer;
                const uint32_t slots = task.end > task.first ? (task.end - task.first + 15) / 16 : 0;
                uint32_t page0 = 0, page1 = 0;
                for (uint32_t x = 0; x < slots; ++x) {
                    if ((x & 31) == 0) {
                        const uint32_t token = task.first + (x + lane) * 16;
                        if (x + lane < slots) {
                            // (the first half may lie before everything that is visible, the second behind it)
                            const bool low = token + 8 > task.begin || token + 8 >= task.end;
                            page0 = p.page_ids[table + ((low ? token : token + 8) >> page_shift)];
                            page1 = page_shift == 3 && low && token + 8 < task.end ? p.page_ids[table + ((token + 8) >> page_shift)] : page0;
                            if (page0 >= p.pool_pages || page1 >= p.pool_pages) {
                                atomicOr(p.status, kStatusPageOutOfPool);  // nothing outside the pool is read
                                if (page0 >= p.pool_pages) page0 = 0;
                                if (page1 >= p.pool_pages) page1 = 0;
                            }
                        }
                    }
                    const uint32_t first_page = __shfl_sync(0xffffffffu, page0, int(x & 31)), second_page = __shfl_sync(0xffffffffu, page1, int(x & 31));
                    const uint32_t slot = issued % G::kRawSlots, phase = (issued / G::kRawSlots) & 1;
                    if (lane == 0) {
                        ok = mbar_wait(raw_empty + 8 * slot, phase ^ 1, abort_flag, p);
                        if (ok) {
                            const uint32_t bar = raw_full + 8 * slot, dst = smem_addr(raw_ring) + slot * G::kRawBytes;
                            const uint32_t sdst = smem_addr(raw_scales) + slot * 32;
                            const uint32_t row = (task.kv_head << page_shift) + ((task.first + x * 16) & (p.tokens_per_page - 1));
                            mbar_arrive_expect_tx(bar, G::kRawBytes + 32);
                            const uint64_t scales = uint64_t((p.num_kv_heads * 2) << page_shift) * D + ((task.kv_head * 2) << page_shift);
                            tma_load_5d(dst, &kv_map, int32_t(row), int32_t(first_page), bar, policy);
                            if (page_shift == 3) {
                                tma_load_5d(dst + G::kRawBytes / 2, &kv_map, int32_t(row), int32_t(second_page), bar, policy);
                                bulk_load(sdst, p.kv_pages + uint64_t(first_page) * p.page_bytes + scales, 16, bar);
                                bulk_load(sdst + 16, p.kv_pages + uint64_t(second_page) * p.page_bytes + scales, 16, bar);
                            } else {
                                bulk_load(sdst, p.kv_pages + uint64_t(first_page) * p.page_bytes + scales, 32, bar);
                            }
                        }
                    }
                    ++issued;
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) return;
                }
            };
            for (uint64_t index = blockIdx.x; index < total && ok; index += gridDim.x) {
                const uint32_t cell = uint32_t(index / pairs), pair = pairs - 1 - uint32_t(index % pairs);
                ScaledTcTask task{};
                task.kv_head = cell / p.head_ranges;
                const uint32_t skipped = (cell % p.head_ranges) * p.heads_per_task;
                task.head_begin = task.kv_head * p.group + skipped;
                task.num_heads = min(p.heads_per_task, p.group - skipped);
                // two tiles of one request that begin together; else one after the other
                const bool first = decode(stride * pair, 0, task);
                const bool together = first && stride == 2 && decode(2 * pair + 1, 1, task) && task.kv_begin[0] == task.kv_begin[1];
                task.active_b = together ? 1 : 0;
                if (first) stream(task);
                if (!together && stride == 2) {
                    task.active_b = 0;
                    if (decode(2 * pair + 1, 0, task)) stream(task);
                }
            }
            ScaledTcTask last{};
            last.done = 1;
            stream(last);
            if (*abort_flag && lane == 0) {
                // copies already issued may still be landing
                for (uint32_t back = 0; back < uint32_t(G::kRawSlots) && back < issued; ++back) {
                    const uint32_t c = issued - 1 - back;
                    for (uint32_t i = 0; i < p.wait_limit; ++i) {
                        if (mbar_try_wait(raw_full + 8 * (c % G::kRawSlots), (c / G::kRawSlots) & 1)) break;
                    }
                }
            }
        } else if (warp == 15) {
            // ------------------------------ tensor-core issue (one thread) -------------------------------------------
            if (lane == 0) {
                constexpr uint32_t kFormat = umma_format<T>();
                constexpr uint32_t idesc_qk = (1u << 4) | (kFormat << 7) | (kFormat << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
                constexpr uint32_t idesc_pv = idesc_qk | (1u << 16);  // B (V) is stored with the head dimension innermost
                const uint64_t k_desc0 = umma_smem_desc(0, 16, 1024);
                const uint64_t v_desc0 = umma_smem_desc(0, G::kHalfBytes, 1024);
                const uint32_t q_addr = smem_addr(q_tile), k_addr = smem_addr(k_ring), v_addr = smem_addr(v_ring);
                uint32_t k_step = 0, v_step = 0;        // running step numbers of the rings
                uint32_t p_count[2] = {0, 0}, pv_count[2] = {0, 0}, q_count[2] = {0, 0}, o_count[2] = {0, 0};
                bool ok = true;
                auto qk = [&](uint32_t tile) {
                    tmem_fence_after();
                    const uint64_t q = k_desc0 + uint64_t((q_addr + tile * G::kOperandBytes) >> 4);
                    const uint64_t k = k_desc0 + uint64_t((k_addr + (k_step & 1) * G::kOperandBytes) >> 4);
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        const uint64_t at = uint64_t(((kk / 4) * G::kHalfBytes + (kk % 4) * 32) >> 4);
                        umma_ss(tmem_s + 128 * tile, q + at, k + at, idesc_qk, kk > 0 ? 1u : 0u);
                    }
                    umma_commit(s_full + 8 * tile);
                };
                for (uint32_t taken = 0; ok; ++taken) {
                    const uint32_t ts = taken & 1;
                    if (!mbar_wait(task_full + 8 * ts, (taken >> 1) & 1, abort_flag, p)) break;
                    if (tasks[ts].done) break;
                    const uint32_t steps = tasks[ts].steps, tiles = 1 + tasks[ts].active_b;
                    mbar_arrive(task_empty + 8 * ts);
                    for (uint32_t j = 0; j <= steps && ok && steps > 0; ++j) {
                        // products of step j - 1 with V, then scores of step j; tile by tile
                        if (j < steps) ok = mbar_wait(k_full + 8 * (k_step & 1), (k_step >> 1) & 1, abort_flag, p);
                        for (uint32_t tile = 0; tile < tiles && ok; ++tile) {
                            if (j > 0) {
                                ok = mbar_wait(p_full + 8 * tile, p_count[tile] & 1, abort_flag, p);
                                ++p_count[tile];
                                if (ok && tile == 0) ok = mbar_wait(v_full + 8 * (v_step & 1), (v_step >> 1) & 1, abort_flag, p);
                                if (ok && j == 1) {
                                    // the tile's first product overwrites O: its last epilogue must have read it
                                    ok = mbar_wait(o_free + 8 * tile, (o_count[tile] & 1) ^ 1, abort_flag, p);
                                    ++o_count[tile];
                                }
                                if (!ok) break;
                                tmem_fence_after();
                                const bool with_remainder = kRemainder && (remainder_flag[4 * tile] | remainder_flag[4 * tile + 1] |
                                                                           remainder_flag[4 * tile + 2] | remainder_flag[4 * tile + 3]) != 0u;
                                const uint64_t v = v_desc0 + uint64_t((v_addr + (v_step & 1) * G::kOperandBytes) >> 4);
                                const uint32_t probabilities = tmem_s + 128 * tile;
#pragma unroll
                                for (int i = 0; i < G::kStep / 16; ++i) {
                                    umma_ts(tmem_o + 128 * tile, probabilities + 8 * i, v + uint64_t((i * 2048) >> 4), idesc_pv, j > 1 || i > 0 ? 1u : 0u);
                                }
                                if (with_remainder) {
#pragma unroll
                                    for (int i = 0; i < G::kStep / 16; ++i) {
                                        umma_ts(tmem_o + 128 * tile, probabilities + 64 + 8 * i, v + uint64_t((i * 2048) >> 4), idesc_pv, 1u);
                                    }
                                }
                                umma_commit(pv_done + 8 * tile);
                                if (tile + 1 == tiles) umma_commit(v_empty + 8 * (v_step & 1));
                                if (j == steps) umma_commit(o_full + 8 * tile);
                            }
                            if (j < steps) {
                                if (j == 0) {
                                    ok = mbar_wait(q_full + 8 * tile, q_count[tile] & 1, abort_flag, p);
                                    ++q_count[tile];
                                } else {
                                    // the scores go where the probabilities of the product before lie
                                    ok = mbar_wait(pv_done + 8 * tile, pv_count[tile] & 1, abort_flag, p);
                                }
                                if (!ok) break;
                                qk(tile);
                            }
                            if (j > 0) ++pv_count[tile];
                        }
                        if (!ok) break;
                        if (j < steps) {
                            umma_commit(k_empty + 8 * (k_step & 1));
                            ++k_step;
                        }
                        if (j > 0) ++v_step;
                    }
                }
                // nothing issued here may still be running when tensor memory is freed (bounded, also on the abort path)
                umma_commit(drain);
                for (uint32_t i = 0; i < p.wait_limit; ++i) {
                    if (mbar_try_wait(drain, 0)) break;
                }
            }
        } else {
            // ------------------------------ conversion ---------------------------------------------------------------
            // A warp takes every kConverters-th 16-token chunk. Eight consecutive lanes take the lower four 16-byte pieces
            // of one row and the upper four of its neighbour: that makes their loads, and both rounds of their 16-byte
            // stores, touch every bank once (128-byte swizzle on both sides).
            const uint32_t sub = (lane >> 2) & 1, cc = lane & 3, row_pair = lane >> 4, flip = (lane >> 3) & 1;
            const uint32_t row4 = 2 * row_pair + (sub ^ flip), piece = 4 * sub + cc;
            const bool short_pages = p.tokens_per_page == 8;
            uint32_t step = 0, raw = 0, chunk_number = 0;  // running numbers
            bool ok = true;
            for (uint32_t taken = 0; ok; ++taken) {
                const uint32_t ts = taken & 1;
                if (!mbar_wait_warp(task_full + 8 * ts, (taken >> 1) & 1, abort_flag, p)) break;
                if (tasks[ts].done) break;
                const uint32_t steps = tasks[ts].steps, first = tasks[ts].first, begin = tasks[ts].begin, end = tasks[ts].end;
                __syncwarp();
                if (lane == 0) mbar_arrive(task_empty + 8 * ts);
                const uint32_t slots = end > first ? (end - first + 15) / 16 : 0;
                for (uint32_t j = 0; j < steps && ok; ++j, ++step) {
                    const uint32_t stage = step & 1, phase = (step >> 1) & 1;
                    for (uint32_t c = 0; c < uint32_t(G::kChunks); ++c, ++chunk_number) {
                        const uint32_t x = j * G::kChunks + c;
                        const uint32_t raw_number = raw + x;
                        if (chunk_number % G::kConverters != warp - 8) continue;
                        const bool there = x < slots;
                        const uint32_t slot = raw_number % G::kRawSlots;
                        if (there) ok = mbar_wait_warp(raw_full + 8 * slot, (raw_number / G::kRawSlots) & 1, abort_flag, p);
                        const uint8_t* const source = raw_ring + slot * G::kRawBytes;
                        const uint8_t* const scales = raw_scales + slot * 32;
#pragma unroll
                        for (int plane = 0; plane < 2; ++plane) {
                            ok = ok && mbar_wait_warp((plane == 0 ? k_empty : v_empty) + 8 * stage, phase ^ 1, abort_flag, p);
                            if (!ok) break;
                            uint8_t* const out = (plane == 0 ? k_ring : v_ring) + stage * G::kOperandBytes + (piece >> 2) * G::kHalfBytes;
                            uint4 words[4];
                            uint32_t one[4], two[4];
                            bool large = false;
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const uint32_t row = 4 * i + row4;
                                words[i] = make_uint4(0, 0, 0, 0);
                                uint32_t b = 0;
                                const uint32_t token = first + x * 16 + row;
                                if (there && token >= begin && token < end) {
                                    // (a copy holds [K/V][16 rows], or two of [K/V][8 rows]; scale bytes alike)
                                    const uint32_t at = short_pages ? (row >> 3) * (G::kRawBytes / 2) + plane * 1024 + (row & 7) * 128
                                                                    : uint32_t(plane) * 2048 + row * 128;
                                    words[i] = *reinterpret_cast<const uint4*>(source + at + ((piece ^ (row & 7)) << 4));
                                    b = scales[short_pages ? (row >> 3) * 16 + plane * 8 + (row & 7) : plane * 16 + row];
                                }
                                scaled_factors<T>(b, plane == 1, one[i], two[i]);
                                large = large || (b >= 134 && b < 255);  // 2^7: E4M3 codes reach 448
                            }
                            const bool saturate = std::is_same<T, __half>::value && __any_sync(0xffffffffu, large);
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const uint32_t row = 4 * i + row4;
                                const uint32_t raw_words[4] = {words[i].x, words[i].y, words[i].z, words[i].w};
                                uint32_t r[8];
#pragma unroll
                                for (int w = 0; w < 4; ++w) {
                                    codes4_to<T, CODE>(raw_words[w], r[2 * w], r[2 * w + 1]);
#pragma unroll
                                    for (int e = 0; e < 2; ++e) {
                                        uint32_t& v = r[2 * w + e];
                                        v = mul2<T>(v, one[i]);
                                        if constexpr (std::is_same<T, __half>::value) {
                                            v = mul2<T>(v, two[i]);
                                            if (saturate) {
                                                // (2^16 is the one value past f16's largest that a code of an f16 row stands for; NaN stays)
                                                const __half2 most = __floats2half2_rn(65504.0f, 65504.0f), least = __floats2half2_rn(-65504.0f, -65504.0f);
                                                const __half2 cut = __hmin2_nan(__hmax2_nan(*reinterpret_cast<__half2*>(&v), least), most);
                                                v = *reinterpret_cast<const uint32_t*>(&cut);
                                            }
                                        }
                                    }
                                }
                                const uint32_t out_row = c * 16 + row;
                                const uint32_t position = (2 * cc) ^ (out_row & 7);
                                *reinterpret_cast<uint4*>(out + out_row * 128 + position * 16) = make_uint4(r[0], r[1], r[2], r[3]);
                                *reinterpret_cast<uint4*>(out + out_row * 128 + (position ^ 1) * 16) = make_uint4(r[4], r[5], r[6], r[7]);
                            }
                            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                            __syncwarp();
                            if (lane == 0) mbar_arrive((plane == 0 ? k_full : v_full) + 8 * stage);
                        }
                        if (!ok) break;
                        if (there && lane == 0) mbar_arrive(raw_empty + 8 * slot);
                    }
                }
                raw += slots;
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
        // ------------------------------ softmax and epilogue of one tile: a thread per row ----------------------------
        const uint32_t tile = warp / 4, quad = warp % 4;
        const uint32_t row = quad * 32 + lane;
        const uint32_t lane_base = (quad * 32) << 16;
        const uint32_t s_at = tmem_s + 128 * tile + lane_base, o_at = tmem_o + 128 * tile + lane_base;
        uint32_t s_count = 0, o_count = 0;
        bool ok = true;
        for (uint32_t taken = 0; ok; ++taken) {
            const uint32_t ts = taken & 1;
            if (!mbar_wait_warp(task_full + 8 * ts, (taken >> 1) & 1, abort_flag, p)) break;
            if (tasks[ts].done) break;
            const ScaledTcTask& task = tasks[ts];
            const bool here = tile == 0 || task.active_b != 0;
            const uint32_t steps = task.steps, first = task.first;
            const uint32_t row_tok = row / p.heads_per_task, row_head = row % p.heads_per_task;
            const bool valid = here && row_tok < task.num_toks[tile] && row_head < task.num_heads;
            const uint32_t head = task.head_begin + row_head, tmpl = task.tmpl[tile];
            const uint64_t q_row = (uint64_t(task.tok_begin[tile]) + row_tok) * p.num_q_heads + head;
            uint32_t lo = 0, hi = 0;
            if (valid) {
                scaled_visible(p, task.tok_begin[tile], row_tok, p.templates[uint64_t(tmpl) * 3 + 1], p.templates[uint64_t(tmpl) * 3 + 2], lo, hi);
                if (hi < lo) hi = lo;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(task_empty + 8 * ts);  // the descriptor has been read
            if (!here) continue;
            if (steps > 0) {
                // the row's Q into its tile (the tile's last product with the Q before has completed: its scores were read)
                uint8_t* const dst = q_tile + tile * G::kOperandBytes + row * 128;
                const uint4* const src = reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + q_row * D);
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                    const uint4 v = valid ? src[c] : make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint4*>(dst + (c / 8) * G::kHalfBytes + (((c % 8) ^ (row & 7)) << 4)) = v;
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full + 8 * tile);
            }
            float m = -INFINITY, l = 0.0f;  // m: raw dot products
            for (uint32_t j = 0; j < steps; ++j) {
                ok = mbar_wait_warp(s_full + 8 * tile, s_count & 1, abort_flag, p);
                ++s_count;
                if (!ok) break;
                tmem_fence_after();
                uint32_t s[G::kStep];
#pragma unroll
                for (int c = 0; c < G::kStep; c += 32) tmem_ld32(*reinterpret_cast<uint32_t(*)[32]>(&s[c]), s_at + c);
                tmem_ld_wait();
                const uint32_t tok = first + j * G::kStep;
                float top = -INFINITY;
                if (__any_sync(0xffffffffu, tok < lo || tok + G::kStep > hi)) {
#pragma unroll
                    for (int c = 0; c < G::kStep; ++c) {
                        if (!(tok + c >= lo && tok + c < hi)) s[c] = 0xff800000u;  // -inf
                        top = fmaxf(top, __uint_as_float(s[c]));
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < G::kStep; ++c) top = fmaxf(top, __uint_as_float(s[c]));
                }
                // lazy maximum: moved (with the sum and O) only when the step exceeds it by more than 2^8
                const bool grow = top > -INFINITY && (m == -INFINITY || (top - m) * p.scale_log2e > kRescaleLog2);
                if (__any_sync(0xffffffffu, grow)) {
                    const float keep = grow && m != -INFINITY ? fast_exp2((m - top) * p.scale_log2e) : 1.0f;
                    if (grow) {
                        l *= keep;
                        m = top;
                    }
                    if (j > 0) {  // (the commit behind the scores covers the products before them: O is at rest)
#pragma unroll
                        for (int c = 0; c < D; c += 32) {
                            uint32_t o[32];
                            tmem_ld32(o, o_at + c);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
                            tmem_st32(o_at + c, o);
                        }
                        tmem_st_wait();
                    }
                }
                const float shift = m == -INFINITY ? 0.0f : -m * p.scale_log2e;
                // The remainder of a bf16 probability is 2^-9 of it at most. Where the row's sum so far is 64 times the
                // step's largest probability, dropping the step's remainders changes the output by less than 2^-9 / 8 of a
                // V element; the product is left out when that holds for all rows of the tile.
                bool remainder = false;
                if constexpr (kRemainder) {
                    const float most = top == -INFINITY ? 0.0f : fast_exp2(fmaf(top, p.scale_log2e, shift));
                    remainder = __any_sync(0xffffffffu, valid && most * 64.0f > l);
                    if (lane == 0) remainder_flag[4 * tile + quad] = remainder ? 1u : 0u;
                }
                float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
                for (int c = 0; c < G::kStep; c += 32) {
                    uint32_t packed[16], rest[kRemainder ? 16 : 1];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float p0 = fast_exp2(fmaf(__uint_as_float(s[c + 2 * i]), p.scale_log2e, shift));
                        const float p1 = fast_exp2(fmaf(__uint_as_float(s[c + 2 * i + 1]), p.scale_log2e, shift));
                        sum0 += p0;
                        sum1 += p1;
                        packed[i] = pack2<T>(p0, p1);
                        if constexpr (kRemainder) {
                            rest[i] = 0u;
                            if (remainder) {
                                const float2 r = unpack2<T>(packed[i]);
                                rest[i] = pack2<T>(p0 - r.x, p1 - r.y);
                            }
                        }
                    }
                    tmem_st16(s_at + c / 2, packed);
                    // (zeros where another warp of the tile may ask for the second product)
                    if constexpr (kRemainder) tmem_st16(s_at + 64 + c / 2, rest);
                }
                l += sum0 + sum1;
                tmem_st_wait();
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + 8 * tile);
            }
            if (!ok) break;
            // ---- epilogue
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // (a NaN sum stays NaN)
            const uint64_t index = (uint64_t(tmpl) * p.num_q_heads + head) * p.max_q_tokens + row_tok;
            if (steps > 0) {
                ok = mbar_wait_warp(o_full + 8 * tile, o_count & 1, abort_flag, p);
                ++o_count;
                if (!ok) break;
                tmem_fence_after();
            }
#pragma unroll
            for (int c = 0; c < D; c += 32) {
                uint32_t o[32];
                if (steps > 0) {
                    tmem_ld32(o, o_at + c);
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0u;
                }
                if (valid && p.direct != 0) {
                    T* const dst = static_cast<T*>(p.out) + q_row * D + c;
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        uint4 v;
                        v.x = pack2<T>(__uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv);
                        v.y = pack2<T>(__uint_as_float(o[i + 2]) * inv, __uint_as_float(o[i + 3]) * inv);
                        v.z = pack2<T>(__uint_as_float(o[i + 4]) * inv, __uint_as_float(o[i + 5]) * inv);
                        v.w = pack2<T>(__uint_as_float(o[i + 6]) * inv, __uint_as_float(o[i + 7]) * inv);
                        *reinterpret_cast<uint4*>(dst + i) = v;
                    }
                } else if (valid) {
                    float* const dst = p.partial_out + index * D + c;
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        *reinterpret_cast<float4*>(dst + i) = make_float4(__uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv,
                                                                          __uint_as_float(o[i + 2]) * inv, __uint_as_float(o[i + 3]) * inv);
                    }
                }
            }
            if (valid && p.direct == 0) {
                p.partial_sum[index] = l;
                // natural-log domain; a NaN sum needs a finite maximum to reach the merged output
                p.partial_max[index] = m > -INFINITY ? m * (p.scale_log2e * 0.6931471805599453f) : (l == l ? -INFINITY : 0.0f);
            }
            if (steps > 0) {
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(o_free + 8 * tile);
            }
        }
    }
    tmem_fence_before();
    __syncthreads();
    if (warp == 0) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

}  // namespace kh
