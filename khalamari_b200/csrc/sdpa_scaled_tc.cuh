// Attention over scaled 8-bit pages (scaled_kv.cuh) for wide Q tiles (prefill, up to 128 rows a task) on the
// 5th-generation tensor cores.
//
//   S = Q K^T    tcgen05.mma kind::f16, M = 128 rows, N = 64 tokens; Q and K in shared memory, S in tensor memory.
//   O += P V     P from tensor memory (over the columns of the S it came from), V in shared memory, O in tensor memory.
//
// Codes become 16-bit operands of the Q/output type once per step of 64 tokens, in shared memory, with their row's
// power-of-two scale already applied: int8 and E4M3 codes times 2^e are exact in bf16, and in f16 as far as its range goes
// (results are rounded below 2^-14 and saturate at 65504, as values of an f16 cache would). Operands are finite where the
// cache is: a hidden token's probability is 0, and 0 times an infinity would not be. So bf16 operands are 2^-10 of their size
// (2^128, what codes of bf16's largest value stand for, is beyond its range), which the scale of the scores and the epilogue
// take back; it also keeps O, a sum of up to 2^8 |v| for each token, inside f32 for such rows. At head_dim 128 two Q tiles of
// the same sequence and KV head share every converted step (at 256 tensor memory holds the output of one). A probability
// is rounded to the Q/output type: in bf16 that is off by at most 2^-8, no more than what the cache rounds off a V element
// (2^-8 to 2^-7 of the row's largest).
//
// Each tile has two score buffers, so that the scores of step j + 1 are computed while the softmax of step j runs. (With
// one buffer of 128 tokens a tile the loop softmax -> P V -> Q K^T -> softmax was a chain of 7,200 cycles a step, 3,300 of
// them waiting.) A step of two tiles then takes 2,400 cycles at head_dim 128: a softmax warp spends 500 on loading and the
// maximum, 1,050 on the exponentials (the special-function unit's share is 512 a tile, 1,024 for both), 350 waiting for
// scores; the products of both tiles take 1,200, bound by the operands that they read from shared memory. Copies and
// conversion have to keep ahead of that, which takes eight conversion warps (a unit of 16 rows takes 650 cycles, nearly all
// of them latency) and two copy warps (one warp issues a copy and its scale bytes every 660 cycles).
//
// Four sequences of 2,048 new tokens behind contexts of 2,048 to 12,288 (64 / 8 heads, head_dim 128, bf16, int8): 1,740 us
// back to back, 815 TFLOP/s (1,660 us after a pause). No one part bounds it: without the exponentials it is 10 % shorter,
// without the codes' conversion 4 %, without both products 9 %, without all three 34 %; the rest is the hand-over from warp to
// warp in every step. Two of 2,048 behind 4,000 at head_dim 256 (32 / 4 heads): 904 us, 735 TFLOP/s; there the conversion's
// instructions are 14 %, the products 16 %, the exponentials 1 %, and the three together 32 %. 517 tokens at head_dim 256
// (16 / 2 heads, f16, E4M3): 37-39 us with the reduce, of which those parts are 4. (Q rows loaded and O rows stored a row per
// thread: whole rows at a time, with the rows' addresses shuffled, was 5 % slower.)
//
// Warps: softmax and epilogue, one thread a row (0-3 tile A, 4-7 tile B), conversion (8), tensor-core issue (one lane, a
// warp for each tile), task decoding and copies (2). All waits are bounded (mbar_wait); no named barriers between roles.
#pragma once

#include "scaled_kv.cuh"
#include "sdpa_map.cuh"
#include "sdpa_scaled.cuh"
#include "sdpa_tc.cuh"

namespace kh {

template <int D>
struct ScaledTc {
    static_assert(D == 128 || D == 256, "head_dim 128 or 256");
    static constexpr int kTiles = D == 128 ? 2 : 1;              // Q tiles at a time: O takes D columns of tensor memory
    static constexpr int kRows = 128;
    static constexpr int kStep = 64;                             // tokens of a step
    static constexpr int kStages = D == 128 ? 4 : 2;             // steps of K and of V in shared memory
    static constexpr int kChunks = kStep / 16;                   // raw slots (16 tokens) of a step
    static constexpr int kRawSlots = D == 128 ? 8 : 4;
    static constexpr int kLines = D / 128;                       // 128-byte lines of a stored row
    static constexpr int kRawBytes = 2 * 16 * D;
    // a step's K or V, and a Q tile: groups of 64 elements, each [rows][128 bytes] with the 128-byte swizzle
    static constexpr int kGroupBytes = kStep * 128, kOperandBytes = D / 64 * kGroupBytes;
    static constexpr int kQGroupBytes = kRows * 128, kQBytes = D / 64 * kQGroupBytes;
    static constexpr int kSoftmaxWarps = 4 * kTiles;
    // Conversion warps take (chunk, K or V) units in turn. A wait tells a barrier's phases apart by their parity only, and a
    // warp does not wait for every copy, nor do copies land in order; so every slot has two barriers used in turn. Then
    // the phase before the one that a warp waits for belongs to copy r - 2 kRawSlots, which is known to have landed: the
    // warp's last unit was of copy r - 4, by the same copy warp; that copy landed, hence r - kRawSlots had been issued (in
    // order), hence r - 2 kRawSlots had left the slot. (Chunks past the end of a task count as copies: the distance between
    // a warp's units is fixed.)
    static constexpr int kConverters = 8;
    static constexpr int kRawBars = 2 * kRawSlots;
    static_assert(kConverters == 2 * kChunks && kRawSlots % 4 == 0, "a unit of every step, slots of one copy warp");
    static constexpr int kIssueWarp = kSoftmaxWarps + kConverters, kCopyWarp = kIssueWarp + 2;
    static constexpr int kThreads = (kIssueWarp + 4) * 32;
    // The softmax warps need more registers than the launch gives a thread (96 of 640, 128 of 512), the others fewer.
    static constexpr int kSoftmaxRegisters = D == 128 ? 144 : 200, kOtherRegisters = D == 128 ? 64 : 104;
    static constexpr int kRescale = D == 128 ? 16 : 64;          // columns of O scaled at a time, as registers allow
    static_assert(kSoftmaxWarps * kSoftmaxRegisters + (kThreads / 32 - kSoftmaxWarps) * kOtherRegisters <=
                      kThreads / 32 * (65536 / kThreads / 8 * 8), "registers of the launch");
    static constexpr int kSmemBytes = kTiles * kQBytes + 2 * kStages * kOperandBytes + kRawSlots * (kRawBytes + 32) + 1024 + 1024;
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

// Two f32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{ .reg .b64 a, b, c, d; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; mov.b64 c, {%6, %7}; fma.rn.f32x2 d, a, b, c; mov.b64 {%0, %1}, d; }"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{ .reg .b64 a, b, d; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; add.rn.f32x2 d, a, b; mov.b64 {%0, %1}, d; }"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}

template <typename T, int CODE, int D>
__global__ void __launch_bounds__(ScaledTc<D>::kThreads, 1)
sdpa_scaled_tc_kernel(const __grid_constant__ CUtensorMap kv_map, const __grid_constant__ CUtensorMap, const MapParams p) {
    using G = ScaledTc<D>;
    constexpr float kRescaleLog2 = 8.0f;  // O is rescaled only when a row maximum grows by more than 2^8

    extern __shared__ uint8_t smem_raw[];
    uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* const q_tile = smem;                                  // [kTiles]
    uint8_t* const k_ring = smem + G::kTiles * G::kQBytes;         // [kStages]
    uint8_t* const v_ring = k_ring + G::kStages * G::kOperandBytes;
    uint8_t* const raw_ring = v_ring + G::kStages * G::kOperandBytes;  // [kRawSlots]
    uint8_t* const raw_scales = raw_ring + G::kRawSlots * G::kRawBytes;
    ScaledTcTask* const tasks = reinterpret_cast<ScaledTcTask*>(raw_scales + G::kRawSlots * 32);  // [2]
    uint64_t* const bars = reinterpret_cast<uint64_t*>(tasks + 2);
    const uint32_t bar0 = smem_addr(bars);
    const uint32_t raw_empty = bar0;                               // [8]
    const uint32_t k_full = bar0 + 64, k_empty = bar0 + 96, v_full = bar0 + 128, v_empty = bar0 + 160;  // [4] each
    const uint32_t s_full = bar0 + 192, p_full = bar0 + 224;       // [tile][buffer]
    const uint32_t q_full = bar0 + 256, o_full = bar0 + 272, o_free = bar0 + 288, pv_done = bar0 + 304;  // [tile]
    const uint32_t task_full = bar0 + 320, task_empty = bar0 + 336;  // [2]
    const uint32_t drain = bar0 + 352, raw_full = bar0 + 360;      // [1], [16]
    constexpr int kBars = 61;
    volatile uint32_t* const abort_flag = reinterpret_cast<volatile uint32_t*>(bars + kBars);
    uint32_t* const tmem_slot = const_cast<uint32_t*>(abort_flag) + 1;
    static_assert(sizeof(ScaledTcTask) * 2 + kBars * 8 + 16 <= 1024, "small shared memory");

    // (values from a shuffle are known to be the same in a whole warp: what is computed from them stays in uniform registers,
    // where the tensor-core instructions and copies take their operands)
    const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < G::kRawSlots; ++i) {
            mbar_init(raw_empty + 8 * i, 2);  // its K and its V have been converted
        }
        for (int i = 0; i < G::kRawBars; ++i) mbar_init(raw_full + 8 * i, 1);
        for (int i = 0; i < 4; ++i) {
            mbar_init(k_full + 8 * i, G::kChunks);
            mbar_init(v_full + 8 * i, G::kChunks);
            mbar_init(k_empty + 8 * i, G::kTiles);
            mbar_init(v_empty + 8 * i, G::kTiles);
            mbar_init(s_full + 8 * i, 1);
            mbar_init(p_full + 8 * i, 4);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(q_full + 8 * i, 4);
            mbar_init(o_full + 8 * i, 1);
            mbar_init(o_free + 8 * i, 4);
            mbar_init(pv_done + 8 * i, 1);
            mbar_init(task_full + 8 * i, 1);
            mbar_init(task_empty + 8 * i, G::kSoftmaxWarps + G::kConverters + G::kTiles + 1);  // (1: the second copy warp)
        }
        mbar_init(drain, G::kTiles);
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
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    const uint32_t tmem_s = tmem, tmem_o = tmem + 256;  // + 128 * tile (+ 64 * buffer); P over the first half of its S
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const ActiveCounts a = resolve_active(p);

    if (warp >= uint32_t(G::kSoftmaxWarps)) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::kOtherRegisters));
        if (warp >= uint32_t(G::kCopyWarp)) {
            const uint32_t which = warp - G::kCopyWarp;
            // ------------------------------ tasks and copies --------------------------------------------------------
            // Tasks are pairs of neighbouring templates, dealt round robin KV head by KV head, so that at any moment the
            // CTAs read the same K/V rows through L2; within a head from the last template to the first, so that the
            // long rows of a causal batch do not come last.
            const uint32_t cells = p.num_kv_heads * p.head_ranges;
            // (no more tasks than SMs: one tile each; a pair costs about what a single tile does)
            const uint32_t stride = G::kTiles == 2 && uint64_t(a.templates) * cells > gridDim.x ? 2 : 1;
            const uint32_t pairs = (a.templates + stride - 1) / stride;
            const uint64_t total = uint64_t(pairs) * cells;
            const uint32_t page_shift = 31 - __clz(int(p.tokens_per_page));
            const uint64_t policy = l2_evict_first_policy();
            uint32_t published = 0;          // tasks
            uint32_t copied = 0, next = 2 * which;  // running numbers of chunks: of tasks done, of this warp's next pair
            bool ok = true;
            // Two neighbouring templates at once, a half warp each: is there a tile to work on, and for which request.
            auto decode = [&](uint32_t tmpl0, ScaledTcTask& task, uint32_t& slot0, uint32_t& slot1) -> uint32_t {
                const uint32_t tile = lane >> 4, sub = lane & 15, tmpl = tmpl0 + tile;
                uint32_t there = 0, begin = 0, num = 0, slot = 0, lo = 0xffffffffu, hi = 0;
                if (tmpl < a.templates && (tile == 0 || stride == 2)) {
                    const uint32_t range = p.templates[uint64_t(tmpl) * 3];
                    const uint32_t kv_begin = p.templates[uint64_t(tmpl) * 3 + 1], kv_end = p.templates[uint64_t(tmpl) * 3 + 2];
                    uint32_t end = 0;
                    if (p.q_ranges == nullptr) {
                        there = range < a.tokens;
                        begin = range;
                        end = range + 1;
                    } else if (range < a.q_tiles) {
                        begin = p.q_ranges[range * 2];
                        end = p.q_ranges[range * 2 + 1];
                        there = begin < a.tokens && end <= a.tokens && end > begin;
                    }
                    if (there) {
                        num = min(end - begin, p.max_q_tokens);
                        slot = p.req_slots[begin];
                        // what some row of the tile sees
                        for (uint32_t tok = sub; tok < num; tok += 16) {
                            uint32_t l, h;
                            scaled_visible(p, begin, tok, kv_begin, kv_end, l, h);
                            if (h > l) {
                                lo = min(lo, l);
                                hi = max(hi, h);
                            }
                        }
                        if (slot >= p.num_req_slots || (kv_end > kv_begin && (uint64_t(kv_end) + p.tokens_per_page - 1) / p.tokens_per_page >
                                                                                 p.pages_per_request_layer)) {
                            if (sub == 0) atomicOr(p.status, kStatusMetadataOutOfRange);  // the task is dropped, as in decode_task
                            there = 0;
                        }
                    }
                }
#pragma unroll
                for (int d = 8; d >= 1; d >>= 1) {
                    lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, d));
                    hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, d));
                }
                if (hi <= lo) lo = hi = 0;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    task.tmpl[i] = tmpl0 + i;
                    task.tok_begin[i] = __shfl_sync(0xffffffffu, begin, 16 * i);
                    task.num_toks[i] = __shfl_sync(0xffffffffu, num, 16 * i);
                    task.kv_begin[i] = __shfl_sync(0xffffffffu, lo, 16 * i);
                    task.kv_end[i] = __shfl_sync(0xffffffffu, hi, 16 * i);
                }
                slot0 = __shfl_sync(0xffffffffu, slot, 0);
                slot1 = __shfl_sync(0xffffffffu, slot, 16);
                return __shfl_sync(0xffffffffu, there, 0) | (__shfl_sync(0xffffffffu, there, 16) << 1);
            };
            // This CTA's next task, in order. Every other round of the deal runs backwards: tasks next to one another
            // differ little in length.
            uint64_t round = 0;
            bool second_left = false;  // the second tile of the last pair is a task of its own
            uint32_t second_slot = 0;
            ScaledTcTask task{};
            auto next_task = [&]() {
                if (second_left) {
                    second_left = false;
                    task.tmpl[0] = task.tmpl[1];
                    task.tok_begin[0] = task.tok_begin[1];
                    task.num_toks[0] = task.num_toks[1];
                    task.kv_begin[0] = task.kv_begin[1];
                    task.kv_end[0] = task.kv_end[1];
                    task.req_slot = second_slot;
                    task.active_b = 0;
                } else {
                    uint32_t found = 0;
                    while (found == 0) {
                        const uint64_t index = round * gridDim.x + (round & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
                        if (round * gridDim.x >= total) {
                            task.done = 1;
                            task.steps = 0;
                            return;
                        }
                        ++round;
                        if (index >= total) continue;
                        const uint32_t cell = uint32_t(index / pairs), pair = pairs - 1 - uint32_t(index % pairs);
                        task.kv_head = cell / p.head_ranges;
                        const uint32_t skipped = (cell % p.head_ranges) * p.heads_per_task;
                        task.head_begin = task.kv_head * p.group + skipped;
                        task.num_heads = min(p.heads_per_task, p.group - skipped);
                        uint32_t slot0, slot1;
                        found = decode(stride * pair, task, slot0, slot1);
                        second_slot = slot1;
                        task.req_slot = slot0;
                        // two tiles of one request that begin together; else one after the other
                        task.active_b = found == 3 && slot0 == slot1 && task.kv_begin[0] == task.kv_begin[1] ? 1 : 0;
                        second_left = found == 3 && task.active_b == 0;
                        if (found == 2) {
                            task.tmpl[0] = task.tmpl[1];
                            task.tok_begin[0] = task.tok_begin[1];
                            task.num_toks[0] = task.num_toks[1];
                            task.kv_begin[0] = task.kv_begin[1];
                            task.kv_end[0] = task.kv_end[1];
                            task.req_slot = slot1;
                        }
                    }
                }
                task.begin = task.kv_begin[0];
                task.end = task.active_b ? max(task.kv_end[0], task.kv_end[1]) : task.kv_end[0];  // (they begin together)
                task.first = task.begin / 16 * 16;
                task.steps = task.end > task.first ? (task.end - task.first + G::kStep - 1) / G::kStep : 0;
            };
            // Both copy warps run this: each copies every other pair of chunks, and the first one decodes and publishes.
            if (which == 0) next_task();
            while (ok) {
                const uint32_t ts = published & 1;
                const uint32_t bar = which == 0 ? task_empty + 8 * ts : task_full + 8 * ts;
                ok = mbar_wait_warp(bar, ((published >> 1) & 1) ^ (which == 0 ? 1 : 0), abort_flag, p);
                if (!ok) break;
                if (which == 0) {
                    if (lane == 0) {
                        tasks[ts] = task;
                        mbar_arrive(task_full + 8 * ts);
                    }
                    __syncwarp();
                }
                ++published;
                // what streaming needs; the next task is decoded on the way, once the ring is full
                const ScaledTcTask& now = tasks[ts];
                if (__shfl_sync(0xffffffffu, now.done, 0)) break;
                const uint32_t begin = __shfl_sync(0xffffffffu, now.begin, 0), end = __shfl_sync(0xffffffffu, now.end, 0);
                const uint32_t first = __shfl_sync(0xffffffffu, now.first, 0), kv_head = __shfl_sync(0xffffffffu, now.kv_head, 0);
                const uint32_t req_slot = __shfl_sync(0xffffffffu, now.req_slot, 0);
                const uint32_t chunks = __shfl_sync(0xffffffffu, now.steps, 0) * G::kChunks;
                if (which == 1 && lane == 0) mbar_arrive(task_empty + 8 * ts);
                const uint64_t table = (uint64_t(req_slot) * p.num_gqa_layers + p.layer_index) * p.pages_per_request_layer;
                const uint64_t scales = uint64_t((p.num_kv_heads * 2) << page_shift) * D + ((kv_head * 2) << page_shift);
                const uint32_t slots = end > first ? (end - first + 15) / 16 : 0;
                uint32_t page0 = 0, page1 = 0;
                if (which == 0 && slots == 0) next_task();
                for (uint32_t x = 2 * which; x < chunks; x += 4) {
                    if ((x & 31) == 2 * which && (x & ~31u) + lane < slots) {
                        const uint32_t token = first + ((x & ~31u) + lane) * 16;
                        // (the first half may lie before everything that is visible, the second behind it)
                        const bool low = token + 8 > begin || token + 8 >= end;
                        page0 = p.page_ids[table + ((low ? token : token + 8) >> page_shift)];
                        page1 = page_shift == 3 && low && token + 8 < end ? p.page_ids[table + ((token + 8) >> page_shift)] : page0;
                        if (page0 >= p.pool_pages || page1 >= p.pool_pages) {
                            atomicOr(p.status, kStatusPageOutOfPool);  // nothing outside the pool is read
                            if (page0 >= p.pool_pages) page0 = 0;
                            if (page1 >= p.pool_pages) page1 = 0;
                        }
                    }
                    uint32_t first_page[2], second_page[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        first_page[i] = __shfl_sync(0xffffffffu, page0, int((x + i) & 31));
                        second_page[i] = __shfl_sync(0xffffffffu, page1, int((x + i) & 31));
                    }
                    const uint32_t number = copied + x, slot = number % G::kRawSlots, phase = (number / G::kRawSlots) & 1;
                    const uint32_t bar0 = raw_full + 8 * (number % G::kRawBars);
                    ok = __all_sync(0xffffffffu, mbar_wait(raw_empty + 8 * slot, phase ^ 1, abort_flag, p) &&
                                                     mbar_wait(raw_empty + 8 * slot + 8, phase ^ 1, abort_flag, p));
                    if (!ok) break;
                    if (elect_one()) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const uint32_t bar = bar0 + 8 * i;
                            if (x + i < slots) {
                                const uint32_t dst = smem_addr(raw_ring) + (slot + i) * G::kRawBytes, sdst = smem_addr(raw_scales) + (slot + i) * 32;
                                const uint32_t in_page = (first + (x + i) * 16) & (p.tokens_per_page - 1);  // (8-token pages: 0)
                                const int32_t page_row = int32_t((kv_head << page_shift) + in_page);
                                const uint8_t* const s0 = p.kv_pages + uint64_t(first_page[i]) * p.page_bytes + scales + in_page;
                                mbar_arrive_expect_tx(bar, G::kRawBytes + 32);
                                tma_load_5d(dst, &kv_map, page_row, int32_t(first_page[i]), bar, policy);
                                if (page_shift == 3) {
                                    tma_load_5d(dst + G::kRawBytes / 2, &kv_map, page_row, int32_t(second_page[i]), bar, policy);
                                    bulk_load(sdst, s0, 16, bar);
                                    bulk_load(sdst + 16, p.kv_pages + uint64_t(second_page[i]) * p.page_bytes + scales, 16, bar);
                                } else if (page_shift == 4) {
                                    bulk_load(sdst, s0, 32, bar);
                                } else {  // half of a 32-token page: its K and its V bytes
                                    bulk_load(sdst, s0, 16, bar);
                                    bulk_load(sdst + 16, s0 + p.tokens_per_page, 16, bar);
                                }
                            } else {
                                mbar_arrive(bar);  // the last step's chunks past the end: nothing to copy
                            }
                        }
                    }
                    __syncwarp();
                    next = number + 4;
                    if (which == 0 && x == ((min(slots, uint32_t(G::kRawSlots)) - 1) & ~3u)) next_task();
                }
                copied += chunks;
            }
            if (*abort_flag && lane == 0) {
                // copies already issued may still be landing
                for (uint32_t c = next; c >= 4 && c + G::kRawSlots > next;) {
                    c -= 4;
                    for (uint32_t n = c; n < c + 2; ++n) {
                        for (uint32_t i = 0; i < p.wait_limit; ++i) {
                            if (mbar_try_wait(raw_full + 8 * (n % G::kRawBars), (n / G::kRawBars) & 1)) break;
                        }
                    }
                }
            }
        } else if (warp >= uint32_t(G::kIssueWarp)) {
            // ------------------------------ tensor-core issue: a warp for each tile, one lane issues ------------------
            const uint32_t tile = warp - G::kIssueWarp;
            if (tile < uint32_t(G::kTiles)) {
                constexpr uint32_t kFormat = umma_format<T>();
                constexpr uint32_t idesc = (1u << 4) | (kFormat << 7) | (kFormat << 10) | ((128u >> 4) << 24);
                constexpr uint32_t idesc_qk = idesc | ((uint32_t(G::kStep) >> 3) << 17);
                constexpr uint32_t idesc_pv = idesc | ((uint32_t(D) >> 3) << 17) | (1u << 16);  // V: head dimension innermost
                const uint64_t k_desc0 = umma_smem_desc(0, 16, 1024);
                const uint64_t v_desc0 = umma_smem_desc(0, G::kGroupBytes, 1024);
                const uint64_t q_desc = k_desc0 + uint64_t((smem_addr(q_tile) + tile * G::kQBytes) >> 4);
                const uint32_t k_addr = smem_addr(k_ring), v_addr = smem_addr(v_ring);
                const uint32_t scores = tmem_s + 128 * tile, out = tmem_o + 128 * tile;
                uint32_t step = 0;                              // running step number of the K and V rings
                uint32_t mine = 0;                              // running step number of this tile
                uint32_t done_tasks = 0;                        // of this tile
                bool ok = true;
                auto stage_wait = [&](uint32_t bar, uint32_t number) {
                    return mbar_wait_warp(bar + 8 * (number % G::kStages), (number / G::kStages) & 1, abort_flag, p);
                };
                // scores of step `ahead` steps on, into their buffer
                auto issue_scores = [&](uint32_t ahead) {
                    tmem_fence_after();
                    const uint32_t stage = (step + ahead) % G::kStages, buffer = (mine + ahead) & 1;
                    const uint64_t k = k_desc0 + uint64_t((k_addr + stage * G::kOperandBytes) >> 4);
                    if (elect_one()) {
#pragma unroll
                        for (int kk = 0; kk < D / 16; ++kk) {
                            umma_ss(scores + 64 * buffer, q_desc + uint64_t(((kk / 4) * G::kQGroupBytes + (kk % 4) * 32) >> 4),
                                    k + uint64_t(((kk / 4) * G::kGroupBytes + (kk % 4) * 32) >> 4), idesc_qk, kk > 0 ? 1u : 0u);
                        }
                        umma_commit(s_full + 8 * (2 * tile + buffer));
                        umma_commit(k_empty + 8 * stage);
                    }
                    __syncwarp();
                };
                for (uint32_t taken = 0; ok; ++taken) {
                    const uint32_t ts = taken & 1;
                    if (!mbar_wait_warp(task_full + 8 * ts, (taken >> 1) & 1, abort_flag, p)) break;
                    if (__shfl_sync(0xffffffffu, tasks[ts].done, 0)) break;
                    const uint32_t steps = __shfl_sync(0xffffffffu, tasks[ts].steps, 0);
                    const bool here = tile == 0 || __shfl_sync(0xffffffffu, tasks[ts].active_b, 0) != 0;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(task_empty + 8 * ts);
                    if (!here) {
                        // the steps pass by: this warp's arrivals on their slots
                        for (uint32_t j = 0; j < steps && ok; ++j, ++step) {
                            ok = stage_wait(k_full, step) && stage_wait(v_full, step);
                            if (ok && lane == 0) {
                                mbar_arrive(k_empty + 8 * (step % G::kStages));
                                mbar_arrive(v_empty + 8 * (step % G::kStages));
                            }
                        }
                        continue;
                    }
                    if (steps == 0) continue;
                    ok = mbar_wait_warp(q_full + 8 * tile, done_tasks & 1, abort_flag, p) && stage_wait(k_full, step);
                    if (!ok) break;
                    // (both buffers are free: every product of the task before has been waited for)
                    issue_scores(0);
                    if (steps > 1) {
                        ok = stage_wait(k_full, step + 1);
                        if (!ok) break;
                        issue_scores(1);
                    }
                    for (uint32_t j = 0; j < steps && ok; ++j, ++step, ++mine) {
                        // step j: the product with V, then the scores of step j + 2, which go where its probabilities lie
                        const uint32_t buffer = mine & 1;
                        ok = mbar_wait_warp(p_full + 8 * (2 * tile + buffer), (mine >> 1) & 1, abort_flag, p) && stage_wait(v_full, step);
                        // the tile's first product overwrites O: its last epilogue must have read it
                        if (ok && j == 0) ok = mbar_wait_warp(o_free + 8 * tile, (done_tasks & 1) ^ 1, abort_flag, p);
                        if (!ok) break;
                        tmem_fence_after();
                        const uint32_t stage = step % G::kStages;
                        const uint64_t v = v_desc0 + uint64_t((v_addr + stage * G::kOperandBytes) >> 4);
                        if (elect_one()) {
#pragma unroll
                            for (int i = 0; i < G::kStep / 16; ++i) {
                                umma_ts(out, scores + 64 * buffer + 8 * i, v + uint64_t((i * 2048) >> 4), idesc_pv, j > 0 || i > 0 ? 1u : 0u);
                            }
                            umma_commit(pv_done + 8 * tile);
                            umma_commit(v_empty + 8 * stage);
                            if (j + 1 == steps) umma_commit(o_full + 8 * tile);
                        }
                        __syncwarp();
                        if (j + 2 < steps) ok = stage_wait(k_full, step + 2);
                        ok = ok && mbar_wait_warp(pv_done + 8 * tile, mine & 1, abort_flag, p);
                        if (!ok) break;
                        if (j + 2 < steps) issue_scores(2);
                    }
                    ++done_tasks;
                }
                // nothing issued here may still be running when tensor memory is freed (bounded, also on the abort path)
                if (elect_one()) umma_commit(drain);
                __syncwarp();
                for (uint32_t i = 0; i < p.wait_limit; ++i) {
                    if (mbar_try_wait(drain, 0)) break;
                }
            }
        } else {
            // ------------------------------ conversion ---------------------------------------------------------------
            // A warp takes every kConverters-th unit: the K or the V rows of a 16-token chunk. Eight consecutive lanes take the
            // lower four 16-byte pieces of one row and the upper four of its neighbour: that makes their loads, and both
            // rounds of their 16-byte stores, touch every bank once (128-byte swizzle on both sides).
            const uint32_t sub = (lane >> 2) & 1, cc = lane & 3, row_pair = lane >> 4, flip = (lane >> 3) & 1;
            const uint32_t row4 = 2 * row_pair + (sub ^ flip), piece = 4 * sub + cc;
            // Rows 4 i + row4, i < 4. A copy holds [K/V][line][16 rows], or two of [K/V][line][8 rows] (8-token pages); scale
            // bytes alike, without lines.
            const bool short_pages = p.tokens_per_page == 8;
            const uint32_t in_lane = row4 * 128 + ((piece ^ row4) << 4);
            const uint32_t out_lane = sub * G::kGroupBytes + row4 * 128 + (((2 * cc) ^ row4) << 4);
            const uint32_t line_stride = short_pages ? 1024 : 2048, half_stride = short_pages ? G::kRawBytes / 2 : 1024;
            const uint32_t scale_plane = short_pages ? 8 : 16, scale_half = short_pages ? 16 : 8;
            uint32_t step = 0;  // running number
            bool ok = true;
            for (uint32_t taken = 0; ok; ++taken) {
                const uint32_t ts = taken & 1;
                if (!mbar_wait_warp(task_full + 8 * ts, (taken >> 1) & 1, abort_flag, p)) break;
                if (tasks[ts].done) break;
                const uint32_t steps = tasks[ts].steps, first = tasks[ts].first, begin = tasks[ts].begin, end = tasks[ts].end;
                __syncwarp();
                if (lane == 0) mbar_arrive(task_empty + 8 * ts);
                const uint32_t slots = end > first ? (end - first + 15) / 16 : 0;
                const uint32_t units = steps * G::kChunks * 2;
                // (one unit of every step: a warp keeps its chunk of a step and its plane)
                for (uint32_t u = warp - G::kSoftmaxWarps; u < units && ok; u += G::kConverters) {
                    const uint32_t x = u >> 1, plane = u & 1;
                    const uint32_t number = step + x / G::kChunks, stage = number % G::kStages, phase = (number / G::kStages) & 1;
                    const uint32_t raw_number = step * G::kChunks + x, slot = raw_number % G::kRawSlots;
                    const bool there = x < slots;
                    ok = mbar_wait_warp(raw_full + 8 * (raw_number % G::kRawBars), (raw_number / G::kRawBars) & 1, abort_flag, p);
                    const uint8_t* const source = raw_ring + slot * G::kRawBytes;
                    const uint8_t* const scales = raw_scales + slot * 32 + row4;
                    const uint32_t token = first + x * 16;
                    const bool whole = there && token >= begin && token + 16 <= end;
                    uint4 words[G::kLines][4];
                    uint32_t b[4];
                    if (!ok) break;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        b[i] = scales[plane * scale_plane + (i >> 1) * scale_half + (i & 1) * 4];
#pragma unroll
                        for (int line = 0; line < G::kLines; ++line) {
                            const uint32_t at = (plane * G::kLines + line) * line_stride + (i >> 1) * half_stride + (i & 1) * 512;
                            words[line][i] = *reinterpret_cast<const uint4*>(source + at + (in_lane ^ ((i & 1) * 64)));
                        }
                    }
                    // the slot takes its next copy while this one is converted
                    __syncwarp();
                    if (lane == 0) mbar_arrive(raw_empty + 8 * slot);
                    ok = mbar_wait_warp((plane == 0 ? k_empty : v_empty) + 8 * stage, phase ^ 1, abort_flag, p);
                    if (!ok) break;
                    if (!whole) {  // rows that nothing sees may hold anything
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t t = token + 4 * i + row4;
                            if (!there || t < begin || t >= end) {
                                b[i] = 0;
#pragma unroll
                                for (int line = 0; line < G::kLines; ++line) words[line][i] = make_uint4(0, 0, 0, 0);
                            }
                        }
                    }
                    uint8_t* const out = (plane == 0 ? k_ring : v_ring) + stage * G::kOperandBytes + (x % G::kChunks) * 2048;
                    bool cut = false;
                    if constexpr (std::is_same<T, __half>::value) {
                        bool large = false;
#pragma unroll
                        for (int i = 0; i < 4; ++i) large = large || (b[i] >= first_large_byte<T>() && b[i] < 255);
                        cut = __any_sync(0xffffffffu, large);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t one, two;
                        operand_factors<T>(b[i], plane == 1, one, two);
#pragma unroll
                        for (int line = 0; line < G::kLines; ++line) {
                            const uint4 w4 = words[line][i];
                            const uint32_t raw_words[4] = {w4.x, w4.y, w4.z, w4.w};
                            uint32_t r[8];
#pragma unroll
                            for (int w = 0; w < 4; ++w) decode4<T, CODE>(raw_words[w], one, two, r[2 * w], r[2 * w + 1]);
                            if (std::is_same<T, __half>::value && cut) {
                                // (2^16 is the one value past f16's largest that a code of an f16 row stands for)
#pragma unroll
                                for (int w = 0; w < 8; ++w) r[w] = saturate2<T>(r[w]);
                            }
                            // rows 4-7 of an eight-row swizzle period: position bit 2 flips
                            uint8_t* const row = out + line * 2 * G::kGroupBytes + i * 512;
                            *reinterpret_cast<uint4*>(row + (out_lane ^ ((i & 1) * 64))) = make_uint4(r[0], r[1], r[2], r[3]);
                            *reinterpret_cast<uint4*>(row + (out_lane ^ ((i & 1) * 64) ^ 16)) = make_uint4(r[4], r[5], r[6], r[7]);
                        }
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive((plane == 0 ? k_full : v_full) + 8 * stage);
                }
                step += steps;
            }
        }
    } else {
        // ------------------------------ softmax and epilogue of one tile: a thread per row ----------------------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(G::kSoftmaxRegisters));
        const uint32_t tile = warp / 4, quad = warp % 4;
        const uint32_t row = quad * 32 + lane;
        const uint32_t lane_base = (quad * 32) << 16;
        const uint32_t o_at = tmem_o + 128 * tile + lane_base;
        const float scale_log2e = p.scale_log2e * float(1 << kOperandShift<T>);
        uint32_t mine = 0, done_tasks = 0;  // running numbers of this tile: steps, tasks
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
                // the row's Q into its tile (the scores of the tile's last task have all been read: nothing uses it any more)
                uint8_t* const dst = q_tile + tile * G::kQBytes + row * 128;
                const uint4* const src = reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + q_row * D);
#pragma unroll
                for (int c = 0; c < D / 8; ++c) {
                    const uint4 v = valid ? src[c] : make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint4*>(dst + (c / 8) * G::kQGroupBytes + (((c % 8) ^ (row & 7)) << 4)) = v;
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full + 8 * tile);
            }
            float m = -INFINITY, l = 0.0f;  // m: raw dot products
            for (uint32_t j = 0; j < steps; ++j, ++mine) {
                const uint32_t buffer = mine & 1;
                const uint32_t s_at = tmem_s + 128 * tile + 64 * buffer + lane_base;
                ok = mbar_wait_warp(s_full + 8 * (2 * tile + buffer), (mine >> 1) & 1, abort_flag, p);
                if (!ok) break;
                tmem_fence_after();
                uint32_t s[G::kStep];
#pragma unroll
                for (int c = 0; c < G::kStep; c += 32) tmem_ld32(*reinterpret_cast<uint32_t(*)[32]>(&s[c]), s_at + c);
                tmem_ld_wait();
                const uint32_t tok = first + j * G::kStep;
                if (__any_sync(0xffffffffu, tok < lo || tok + G::kStep > hi)) {
#pragma unroll
                    for (int c = 0; c < G::kStep; ++c) {
                        if (!(tok + c >= lo && tok + c < hi)) s[c] = 0xff800000u;  // -inf
                    }
                }
                float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < G::kStep; c += 8) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        tops[i] = fmaxf(fmaxf(tops[i], __uint_as_float(s[c + 2 * i])), __uint_as_float(s[c + 2 * i + 1]));
                    }
                }
                const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
                // lazy maximum: moved (with the sum and O) only when the step exceeds it by more than 2^8
                const bool grow = top > -INFINITY && (m == -INFINITY || (top - m) * scale_log2e > kRescaleLog2);
                if (__any_sync(0xffffffffu, grow)) {
                    const float keep = grow && m != -INFINITY ? fast_exp2((m - top) * scale_log2e) : 1.0f;
                    if (grow) {
                        l *= keep;
                        m = top;
                    }
                    if (j > 0) {
                        // O is at rest once the product of the step before has completed
                        ok = mbar_wait_warp(pv_done + 8 * tile, (mine - 1) & 1, abort_flag, p);
                        if (!ok) break;
                        tmem_fence_after();
#pragma unroll
                        for (int c = 0; c < D; c += G::kRescale) {
                            uint32_t o[G::kRescale];
#pragma unroll
                            for (int i = 0; i < G::kRescale; i += 16) tmem_ld16(*reinterpret_cast<uint32_t(*)[16]>(&o[i]), o_at + c + i);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < G::kRescale; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
#pragma unroll
                            for (int i = 0; i < G::kRescale; i += 16) tmem_st16(o_at + c + i, *reinterpret_cast<uint32_t(*)[16]>(&o[i]));
                        }
                        tmem_st_wait();
                    }
                }
                const float shift = m == -INFINITY ? 0.0f : -m * scale_log2e;
                const float2 scale2 = make_float2(scale_log2e, scale_log2e), shift2 = make_float2(shift, shift);
                float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                for (int c = 0; c < G::kStep; c += 32) {
                    uint32_t packed[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float2 x = fma2(make_float2(__uint_as_float(s[c + 2 * i]), __uint_as_float(s[c + 2 * i + 1])), scale2, shift2);
                        x.x = fast_exp2(x.x);
                        x.y = fast_exp2(x.y);
                        sum[i & 1] = add2(sum[i & 1], x);
                        packed[i] = pack2<T>(x.x, x.y);
                    }
                    tmem_st16(s_at + c / 2, packed);
                }
                l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                tmem_st_wait();
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + 8 * (2 * tile + buffer));
            }
            if (!ok) break;
            // ---- epilogue
            // (a token that is seen adds 1 at the maximum, unless every score is -inf: that softmax is NaN)
            if (l == 0.0f && hi > lo) l = __uint_as_float(0x7fc00000u);
            const float inv = l == 0.0f ? 0.0f : float(1 << kOperandShift<T>) / l;  // (a NaN sum stays NaN)
            const uint64_t index = (uint64_t(tmpl) * p.num_q_heads + head) * p.max_q_tokens + row_tok;
            if (steps > 0) {
                ok = mbar_wait_warp(o_full + 8 * tile, done_tasks & 1, abort_flag, p);
                ++done_tasks;
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
                // (averages of largest values: rounded probabilities can take them a step too far)
                if (valid && p.direct != 0) {
                    T* const dst = static_cast<T*>(p.out) + q_row * D + c;
                    auto pair = [&](int i) { return saturate2<T>(pack2<T>(__uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv)); };
#pragma unroll
                    for (int i = 0; i < 32; i += 8) *reinterpret_cast<uint4*>(dst + i) = make_uint4(pair(i), pair(i + 2), pair(i + 4), pair(i + 6));
                } else if (valid) {
                    float* const dst = p.partial_out + index * D + c;
                    auto one = [&](int i) { return saturate<__nv_bfloat16>(__uint_as_float(o[i]) * inv); };
#pragma unroll
                    for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4*>(dst + i) = make_float4(one(i), one(i + 1), one(i + 2), one(i + 3));
                }
            }
            if (valid && p.direct == 0) {
                publish_partial_stats(p.partial_sum, p.partial_max, index, m * (scale_log2e * 0.6931471805599453f), l);
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
