// KV page read: gathers cached K and V rows into flat [rows][Hkv][D] arrays, the inverse of the page write
// (kv_page_write.cu) for every page element type it stores. Addresses as there; scale bytes as in scaled_kv.cuh.
// HBM-bound: a lane turns eight codes (8 bytes, or 16 of a 16-bit page) into 16 output bytes, so that a warp's loads
// and stores are whole lines; over scaled pages a warp takes a whole row (all heads), four vectors in flight per lane,
// which spreads the address arithmetic that bounded a thread-per-vector form (117,332 rows of 4 x 256: 320 us then, 125 us
// now, 5.7 TB/s; floor 110 us).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <memory>

#include "cuda_objects.h"
#include "scaled_kv.cuh"

namespace kh {

struct PageReadParams {
    const uint8_t* pages;
    uint16_t* flat_k;
    uint16_t* flat_v;
    const uint32_t* req_slots;
    const uint32_t* flat_token_indices;
    const uint32_t* page_ids;
    uint32_t* status;
    uint32_t num_active_token_reads;
    uint32_t layer_index;
    uint32_t num_req_slots;
    uint32_t num_gqa_layers;
    uint32_t num_blocks;
    uint32_t num_page_ids_per_block;
    uint32_t num_kv_heads;
    uint32_t head_dim;
    uint32_t tokens_per_page;
    uint32_t page_bytes;
    uint32_t pool_pages;
};

// What a page stores.
enum PageKind : int { kPage16 = 0, kPageE4M3 = 1 };  // (scaled pages have a kernel of their own)

// E4M3 values are exact in both types.
template <typename T>
__device__ __forceinline__ uint32_t pack_exact(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack_exact<__half>(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack_exact<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// VEC elements per lane: 8, or 1 for rows or buffers that 16-byte accesses do not fit (16-bit and plain FP8 pages of odd
// head dimensions).
template <typename T, int KIND, int VEC>
__global__ void __launch_bounds__(256) kv_page_read_kernel(const PageReadParams p) {
    constexpr int kBytes = KIND == kPage16 ? 2 : 1;
    const uint32_t vecs = p.head_dim / VEC;
    const uint32_t per_read = 2 * p.num_kv_heads * vecs;  // [head][plane][vector]
    const uint64_t total = uint64_t(p.num_active_token_reads) * per_read;
    for (uint64_t gid = uint64_t(blockIdx.x) * blockDim.x + threadIdx.x; gid < total;
         gid += uint64_t(gridDim.x) * blockDim.x) {
        const uint32_t read = uint32_t(gid / per_read);
        uint32_t rest = uint32_t(gid % per_read);
        const uint32_t d = (rest % vecs) * VEC;
        rest /= vecs;
        const uint32_t plane = rest & 1, head = rest >> 1;
        const uint32_t slot = p.req_slots[read];
        const uint32_t token = p.flat_token_indices[read];
        const uint32_t block = token / (p.tokens_per_page * p.num_page_ids_per_block);
        const uint32_t id_in_block = (token / p.tokens_per_page) % p.num_page_ids_per_block;
        if (slot >= p.num_req_slots || block >= p.num_blocks) {  // metadata that points past the page table
            atomicOr(p.status, 4u);
            continue;
        }
        const uint64_t entry =
            ((uint64_t(slot) * p.num_gqa_layers + p.layer_index) * p.num_blocks + block) * p.num_page_ids_per_block +
            id_in_block;
        const uint32_t page = p.page_ids[entry];
        if (page >= p.pool_pages) {
            atomicOr(p.status, 2u);
            continue;
        }
        const uint8_t* const page_base = p.pages + uint64_t(page) * p.page_bytes;
        const uint32_t row = token % p.tokens_per_page;
        const uint64_t elem = ((uint64_t(plane) * p.num_kv_heads + head) * p.tokens_per_page + row) * p.head_dim + d;
        uint16_t* const out = (plane == 0 ? p.flat_k : p.flat_v) + (uint64_t(read) * p.num_kv_heads + head) * p.head_dim + d;
        if constexpr (KIND == kPage16) {
            if constexpr (VEC == 8) *reinterpret_cast<uint4*>(out) = *reinterpret_cast<const uint4*>(page_base + elem * kBytes);
            else *out = *reinterpret_cast<const uint16_t*>(page_base + elem * kBytes);
        } else {
            uint32_t words[(VEC + 3) / 4];
            if constexpr (VEC == 8) {
                const uint2 raw = *reinterpret_cast<const uint2*>(page_base + elem);
                words[0] = raw.x;
                words[1] = raw.y;
            } else {
                words[0] = page_base[elem];
            }
            uint32_t packed[VEC == 8 ? 4 : 1];
#pragma unroll
            for (int w = 0; w < (VEC + 3) / 4; ++w) {
                uint32_t lo, hi;
                codes4_to_half<kCodeE4M3>(words[w], lo, hi);
                const float2 a = __half22float2(*reinterpret_cast<__half2*>(&lo));
                packed[2 * w] = pack_exact<T>(a.x, a.y);
                if constexpr (VEC == 8) {
                    const float2 b = __half22float2(*reinterpret_cast<__half2*>(&hi));
                    packed[2 * w + 1] = pack_exact<T>(b.x, b.y);
                }
            }
            if constexpr (VEC == 8) *reinterpret_cast<uint4*>(out) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
            else *out = uint16_t(packed[0]);
        }
    }
}

template <typename T, int CODE, int D>
__global__ void __launch_bounds__(256) scaled_page_read_kernel(const PageReadParams p) {
    constexpr uint32_t kVecs = D / 8;   // vectors of a row
    constexpr int kFlight = 4;
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t heads = p.num_kv_heads, P = p.tokens_per_page;
    const uint32_t per_plane = heads * kVecs, per_read = 2 * per_plane;
    for (uint64_t unit = (uint64_t(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; unit < p.num_active_token_reads;
         unit += (uint64_t(gridDim.x) * blockDim.x) >> 5) {
        const uint32_t slot = p.req_slots[unit];
        const uint32_t token = p.flat_token_indices[unit];
        const uint32_t block = token / (P * p.num_page_ids_per_block);
        const uint32_t id_in_block = (token / P) % p.num_page_ids_per_block;
        if (slot >= p.num_req_slots || block >= p.num_blocks) {  // metadata that points past the page table
            if (lane == 0) atomicOr(p.status, 4u);
            continue;
        }
        const uint64_t entry =
            ((uint64_t(slot) * p.num_gqa_layers + p.layer_index) * p.num_blocks + block) * p.num_page_ids_per_block +
            id_in_block;
        const uint32_t page = p.page_ids[entry];
        if (page >= p.pool_pages) {
            if (lane == 0) atomicOr(p.status, 2u);
            continue;
        }
        const uint32_t row = token % P;
        const uint8_t* const codes = p.pages + uint64_t(page) * p.page_bytes + uint64_t(row) * D;
        const uint8_t* const scales = p.pages + uint64_t(page) * p.page_bytes + uint64_t(2) * heads * P * D + row;
        for (uint32_t base = lane; base < per_read; base += 32 * kFlight) {
            uint2 raw[kFlight];
            uint32_t b[kFlight];
#pragma unroll
            for (int i = 0; i < kFlight; ++i) {
                const uint32_t vec = base + 32 * i;
                if (vec < per_read) {
                    const uint32_t plane = vec >= per_plane ? 1 : 0, line = vec / kVecs, head = line - plane * heads;  // line = plane * heads + head
                    raw[i] = *reinterpret_cast<const uint2*>(codes + uint64_t(line) * P * D + vec % kVecs * 8);
                    b[i] = scales[(head * 2 + plane) * P];
                }
            }
#pragma unroll
            for (int i = 0; i < kFlight; ++i) {
                const uint32_t vec = base + 32 * i;
                if (vec < per_read) {
                    const uint32_t plane = vec >= per_plane ? 1 : 0;
                    uint32_t one, two, v[4];
                    scaled_factors<T>(b[i], false, one, two);
                    decode4<T, CODE>(raw[i].x, one, two, v[0], v[1]);
                    decode4<T, CODE>(raw[i].y, one, two, v[2], v[3]);
                    if (b[i] >= first_large_byte<T>()) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) v[j] = saturate2<T>(v[j]);
                    }
                    uint16_t* const out = (plane == 0 ? p.flat_k : p.flat_v) + (unit * heads * kVecs + (vec - plane * per_plane)) * 8;
                    *reinterpret_cast<uint4*>(out) = make_uint4(v[0], v[1], v[2], v[3]);
                }
            }
        }
    }
}

template <typename T, int KIND>
static void launch_read(const PageReadParams& p, bool vector, uint32_t blocks, cudaStream_t stream) {
    if (vector) kv_page_read_kernel<T, KIND, 8><<<blocks, 256, 0, stream>>>(p);
    else kv_page_read_kernel<T, KIND, 1><<<blocks, 256, 0, stream>>>(p);
}

template <typename T, int CODE>
static void launch_scaled_read(const PageReadParams& p, uint32_t sm_count, cudaStream_t stream) {
    const uint32_t blocks = std::min<uint32_t>((p.num_active_token_reads + 7) / 8, sm_count * 64);
    if (p.head_dim == 128) scaled_page_read_kernel<T, CODE, 128><<<blocks, 256, 0, stream>>>(p);
    else scaled_page_read_kernel<T, CODE, 256><<<blocks, 256, 0, stream>>>(p);
}

template <typename T>
static void launch_read_kind(const PageReadParams& p, kh_dtype kv_dtype, bool vector, uint32_t sm_count, cudaStream_t stream) {
    if (kv_dtype == KH_DTYPE_INT8_SCALED) return launch_scaled_read<T, kCodeInt8>(p, sm_count, stream);
    if (kv_dtype == KH_DTYPE_FP8_E4M3FN_SCALED) return launch_scaled_read<T, kCodeE4M3>(p, sm_count, stream);
    const uint64_t threads = uint64_t(p.num_active_token_reads) * 2 * p.num_kv_heads * (vector ? p.head_dim / 8 : p.head_dim);
    const uint32_t blocks = uint32_t(std::min<uint64_t>((threads + 255) / 256, uint64_t(sm_count) * 8));
    if (kv_dtype == KH_DTYPE_FP8_E4M3FN) launch_read<T, kPageE4M3>(p, vector, blocks, stream);
    else launch_read<T, kPage16>(p, vector, blocks, stream);
}

}  // namespace kh

using namespace kh;

struct kh_kv_page_read {
    kh_device* device;
    kh_kv_page_read_config config;
    uint32_t tokens_per_page;
};

extern "C" {

kh_status kh_kv_page_read_create(kh_device* device, const kh_kv_page_read_config* config, kh_kv_page_read** out) {
    return guarded([&]() -> kh_status {
        KH_REQUIRE(device && config && out, "null argument");
        auto compute = std::make_unique<kh_kv_page_read>();
        compute->device = device;
        compute->config = *config;
        compute->tokens_per_page = page_write_tokens_per_page(*config);
        *out = compute.release();
        return KH_OK;
    });
}

kh_status kh_kv_page_read_destroy(kh_kv_page_read* compute) {
    delete compute;
    return KH_OK;
}

kh_status kh_kv_page_read_invoke(kh_kv_page_read* compute, kh_stream* stream, const kh_kv_page_read_shape* shape,
                                 const kh_kv_page_read_buffers* buffers, uint32_t num_active_token_reads,
                                 uint32_t page_table_index) {
    return guarded([&]() -> kh_status {
        KH_REQUIRE(compute && stream && shape && buffers, "null argument");
        KH_REQUIRE(stream->device == compute->device, "stream does not belong to the compute's device");
        const kh_kv_page_read_config& c = compute->config;
        const kh_page_table_layout& l = shape->page_table_layout;
        KH_REQUIRE(shape->num_total_token_reads > 0, "GQA KV page read needs token reads");
        KH_REQUIRE(l.num_req_slots > 0 && l.num_blocks > 0 && l.num_gqa_layers > 0 && l.num_page_ids_per_block > 0,
                   "GQA page-table layout dimensions must be positive");
        const uint64_t values = mul_u64(mul_u64(shape->num_total_token_reads, c.num_kv_heads, "GQA KV page-read values"),
                                        c.head_dim, "GQA KV page-read values");
        KH_REQUIRE(num_active_token_reads >= 1 && num_active_token_reads <= shape->num_total_token_reads,
                   "num_active_token_reads %u outside [1, %u]", num_active_token_reads, shape->num_total_token_reads);
        KH_REQUIRE(page_table_index < l.num_gqa_layers, "page_table_index %u out of range", page_table_index);
        need(buffers->flat_k, mul_u64(values, dtype_size(c.dtype), "GQA KV page-read bytes"), "flat_k");
        need(buffers->flat_v, mul_u64(values, dtype_size(c.dtype), "GQA KV page-read bytes"), "flat_v");
        need(buffers->req_slots, uint64_t(shape->num_total_token_reads) * 4, "req_slots");
        need(buffers->flat_token_indices, uint64_t(shape->num_total_token_reads) * 4, "flat_token_indices");
        const uint64_t entries = mul_u64(mul_u64(mul_u64(l.num_req_slots, l.num_gqa_layers, "GQA page-table byte length"),
                                                 l.num_blocks, "GQA page-table byte length"),
                                         l.num_page_ids_per_block, "GQA page-table byte length");
        need(buffers->page_ids, mul_u64(entries, 4, "GQA page-table byte length"), "page_ids");
        need(buffers->pages, c.page_bytes, "pages");
        const bool vector = c.head_dim % 8 == 0 && c.page_bytes % 16 == 0 &&
                            (reinterpret_cast<uintptr_t>(buffers->pages.ptr) & 15) == 0 &&
                            (reinterpret_cast<uintptr_t>(buffers->flat_k.ptr) & 15) == 0 &&
                            (reinterpret_cast<uintptr_t>(buffers->flat_v.ptr) & 15) == 0;
        if (is_scaled(c.kv_dtype)) {
            KH_REQUIRE(vector, "scaled 8-bit pages: pages, flat_k and flat_v must be 16-byte aligned");
        }
        use_device(compute->device);
        PageReadParams p{};
        p.pages = static_cast<const uint8_t*>(buffers->pages.ptr);
        p.flat_k = static_cast<uint16_t*>(buffers->flat_k.ptr);
        p.flat_v = static_cast<uint16_t*>(buffers->flat_v.ptr);
        p.req_slots = static_cast<const uint32_t*>(buffers->req_slots.ptr);
        p.flat_token_indices = static_cast<const uint32_t*>(buffers->flat_token_indices.ptr);
        p.page_ids = static_cast<const uint32_t*>(buffers->page_ids.ptr);
        p.status = compute->device->status;
        p.num_active_token_reads = num_active_token_reads;
        p.layer_index = page_table_index;
        p.num_req_slots = l.num_req_slots;
        p.num_gqa_layers = l.num_gqa_layers;
        p.num_blocks = l.num_blocks;
        p.num_page_ids_per_block = l.num_page_ids_per_block;
        p.num_kv_heads = c.num_kv_heads;
        p.head_dim = c.head_dim;
        p.tokens_per_page = compute->tokens_per_page;
        p.page_bytes = c.page_bytes;
        p.pool_pages = uint32_t(std::min<uint64_t>(buffers->pages.bytes / c.page_bytes, 0xffffffffull));
        if (c.dtype == KH_DTYPE_FLOAT16) launch_read_kind<__half>(p, c.kv_dtype, vector, compute->device->sm_count, stream->stream);
        else launch_read_kind<__nv_bfloat16>(p, c.kv_dtype, vector, compute->device->sm_count, stream->stream);
        KH_CUDA(cudaGetLastError());
        return KH_OK;
    });
}

}  // extern "C"
