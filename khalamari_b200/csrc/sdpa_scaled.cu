// Instances of the attention kernel over scaled 8-bit pages (sdpa_scaled.cuh).
#include <cuda.h>
#include <cuda_runtime.h>

#include "common.h"
#include "map_instance.h"
#include "sdpa_scaled.cuh"

namespace kh {

template <typename T, int CODE, int D, int NQ, int W>
static MapInstance make_scaled_instance() {
    using G = ScaledGeometry<D, NQ, W>;
    return MapInstance{sdpa_scaled_kernel<T, CODE, D, NQ, W>, G::kThreads, G::kSmemBytes, G::kTileTokens, 0, G::kSlots, G::kRows};
}

// Accumulators take D / 16 x NQ x 4 registers of a thread, which sets the warps per SM. Wider tasks are worked on in
// blocks of rows, which read the KV range again (from L2).
template <typename T, int CODE, int D>
static MapInstance pick_scaled_rows(uint32_t rows) {
    if constexpr (D == 128) {
        if (rows <= 8) return make_scaled_instance<T, CODE, 128, 1, 16>();
        if (rows <= 16) return make_scaled_instance<T, CODE, 128, 2, 12>();
        if (rows <= 24) return make_scaled_instance<T, CODE, 128, 3, 8>();
        return make_scaled_instance<T, CODE, 128, 4, 8>();
    } else {
        if (rows <= 8) return make_scaled_instance<T, CODE, 256, 1, 8>();
        if (rows <= 16) return make_scaled_instance<T, CODE, 256, 2, 8>();
        return make_scaled_instance<T, CODE, 256, 3, 8>();
    }
}

template <typename T, int CODE>
static MapInstance pick_scaled_dim(uint32_t head_dim, uint32_t rows) {
    return head_dim == 128 ? pick_scaled_rows<T, CODE, 128>(rows) : pick_scaled_rows<T, CODE, 256>(rows);
}

template <typename T>
static MapInstance pick_scaled_code(kh_dtype kv_dtype, uint32_t head_dim, uint32_t rows) {
    return kv_dtype == KH_DTYPE_INT8_SCALED ? pick_scaled_dim<T, kCodeInt8>(head_dim, rows) : pick_scaled_dim<T, kCodeE4M3>(head_dim, rows);
}

MapInstance pick_instance_scaled(kh_dtype dtype, kh_dtype kv_dtype, uint32_t head_dim, uint32_t rows) {
    KH_REQUIRE(rows >= 1 && rows <= 128, "a Map task holds at most 128 (Q token, Q head) rows (got %u)", rows);
    if (dtype == KH_DTYPE_BFLOAT16) return pick_scaled_code<__nv_bfloat16>(kv_dtype, head_dim, rows);
    KH_REQUIRE(dtype == KH_DTYPE_FLOAT16, "Q/output dtype must be Bfloat16 or Float16 on this backend");
    return pick_scaled_code<__half>(kv_dtype, head_dim, rows);
}

}  // namespace kh
