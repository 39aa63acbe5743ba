// Instances of the attention kernel over scaled 8-bit pages (sdpa_scaled.cuh).
#include <cuda.h>
#include <cuda_runtime.h>

#include "common.h"
#include "map_instance.h"
#include "sdpa_scaled.cuh"
#include "sdpa_scaled_tc.cuh"

namespace kh {

template <typename T, int CODE, int D, int NQ, int W, int HP>
static MapInstance make_stream_instance() {
    using G = ScaledGeometry<D, NQ, W, HP, true>;
    return MapInstance{sdpa_scaled_stream_kernel<T, CODE, D, NQ, W, HP>, G::kThreads, G::kSmemBytes, G::kTileTokens, HP * 16,
                       G::kSlots};
}

template <typename T, int CODE, int D, int NQ, int W>
static MapInstance make_chain_instance() {
    using G = ScaledGeometry<D, NQ, W, 1, false>;
    return MapInstance{sdpa_scaled_chain_kernel<T, CODE, D, NQ, W>, G::kThreads, G::kSmemBytes, G::kTileTokens, 16, G::kSlots};
}

template <typename T, int CODE, int D>
static MapInstance make_tc_instance() {
    using G = ScaledTc<D>;
    return MapInstance{sdpa_scaled_tc_kernel<T, CODE, D>, G::kThreads, G::kSmemBytes, G::kStep, 16, G::kRawSlots};
}

// Accumulators take D / 16 x NQ x 4 registers of a thread, which sets the warps per SM; wider tasks go to tcgen05, whose
// tiles of 128 rows cost the same however few are used (24 rows at head_dim 256: 500 us here, 856 us there). `paired`: the
// KV heads can be taken two at a time (64 decode sequences: 145 us, one at a time 150 us).
template <typename T, int CODE, int D>
static MapInstance pick_scaled_rows(uint32_t rows, bool paired) {
    if (rows > scaled_merging_rows(D)) return make_tc_instance<T, CODE, D>();
    if constexpr (D == 128) {
        if (rows <= 8 && paired) return make_stream_instance<T, CODE, 128, 1, 12, 2>();
        if (rows <= 8) return make_stream_instance<T, CODE, 128, 1, 12, 1>();
        if (rows <= 16) return make_stream_instance<T, CODE, 128, 2, 8, 1>();
        if (rows <= 24) return make_chain_instance<T, CODE, 128, 3, 8>();
        return make_chain_instance<T, CODE, 128, 4, 8>();
    } else {
        if (rows <= 8) return make_stream_instance<T, CODE, 256, 1, 8, 1>();
        if (rows <= 16) return make_chain_instance<T, CODE, 256, 2, 8>();
        return make_chain_instance<T, CODE, 256, 3, 8>();
    }
}

template <typename T, int CODE>
static MapInstance pick_scaled_dim(uint32_t head_dim, uint32_t rows, bool paired) {
    return head_dim == 128 ? pick_scaled_rows<T, CODE, 128>(rows, paired) : pick_scaled_rows<T, CODE, 256>(rows, paired);
}

template <typename T>
static MapInstance pick_scaled_code(kh_dtype kv_dtype, uint32_t head_dim, uint32_t rows, bool paired) {
    return kv_dtype == KH_DTYPE_INT8_SCALED ? pick_scaled_dim<T, kCodeInt8>(head_dim, rows, paired)
                                            : pick_scaled_dim<T, kCodeE4M3>(head_dim, rows, paired);
}

MapInstance pick_instance_scaled(kh_dtype dtype, kh_dtype kv_dtype, uint32_t head_dim, uint32_t tokens_per_page, uint32_t rows, bool paired) {
    KH_REQUIRE(rows >= 1 && rows <= 128, "a Map task holds at most 128 (Q token, Q head) rows (got %u)", rows);
    MapInstance instance;
    if (dtype == KH_DTYPE_BFLOAT16) {
        instance = pick_scaled_code<__nv_bfloat16>(kv_dtype, head_dim, rows, paired);
    } else {
        KH_REQUIRE(dtype == KH_DTYPE_FLOAT16, "Q/output dtype must be Bfloat16 or Float16 on this backend");
        instance = pick_scaled_code<__half>(kv_dtype, head_dim, rows, paired);
    }
    instance.box_rows = instance.box_rows / 16 * int(tokens_per_page < 16 ? tokens_per_page : 16);
    return instance;
}

}  // namespace kh
