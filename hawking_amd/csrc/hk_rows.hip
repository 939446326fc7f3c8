// hk_rows.hip -- row images and the position tiles of a product (hk_rows.h).
#include "hk_rows.h"
#include "hk_rows_image.h"

namespace hk {

// ------------------------------------------------------------------ row images

// Rows of x -> image rows (hk_rows.h), TPR threads a row; the last block makes
// the product's tiles instead.  A row's maximum is taken first: up to four
// chunks a thread stay in registers, more are read again (from the caches).
template <int TYPE, int PLANES, int TPR>
__global__ void __launch_bounds__(256) rows_image_kernel(const void* x, size_t stride, uint32_t n, uint32_t cols, int kind,
                                                         uint32_t chunks, bool vec, RowsWs ws, const int32_t* offsets,
                                                         uint32_t groups, uint32_t n_pos, uint32_t tile_rows,
                                                         uint32_t* status) {
    constexpr int NC = 4;
    __shared__ uint32_t pre[256];
    if (offsets && blockIdx.x == gridDim.x - 1u) {
        rows_tiles(ws, offsets, groups, n_pos, tile_rows, pre);
        return;
    }
    const uint32_t row = blockIdx.x * (256u / TPR) + threadIdx.x / TPR, me = threadIdx.x % TPR;
    if (TPR < 256 && row >= n) return;  // a whole wave
    const size_t base = (size_t)row * stride;
    const uint32_t apart = (kind == HK_BIN || kind == HK_MIXED) ? 16u : 4u;
    auto load = [&](uint32_t ch, float* v) {
        const uint32_t c = rows_chunk_cols(kind, ch).c0;  // columns come in whole 32s
        if (ch < chunks && c < cols) {
            row_load4(TYPE, x, base + c, vec, v);
            row_load4(TYPE, x, base + c + apart, vec, v + 4);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0.0f;
        }
    };
    float v[NC][8];
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < NC; ++i) load(me + (uint32_t)i * TPR, v[i]);
    auto top = [&](const float* e) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            m = fmaxf(m, fabsf(e[i]));
            s += e[i] - e[i];  // NaN for an infinity or a NaN, which fmaxf would drop
        }
        if (s != s) m = INFINITY;
    };
#pragma unroll
    for (int i = 0; i < NC; ++i) top(v[i]);
    for (uint32_t ch = me + NC * TPR; ch < chunks; ch += TPR) {
        float e[8];
        load(ch, e);
        top(e);
    }
    m = wave_max(m);
    if constexpr (TPR == 256) {
        float* red = reinterpret_cast<float*>(pre);
        if ((threadIdx.x & 63u) == 0u) red[threadIdx.x >> 6] = m;
        __syncthreads();
        m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    }
    const bool bad = !isfinite(m);
    int e2 = 0;
    if (!bad && m > 0.0f) (void)frexpf(m, &e2);
    const int E = (!bad && m > 0.0f) ? 14 - e2 : 0;
    if (me == 0) {
        ws.exps[row] = bad ? ROWS_EXP_BAD : E;
        if (bad) atomicOr(status, ROWS_ERR_NONFINITE);
    }
    uint8_t* out = ws.img + (size_t)row * chunks * (16u * PLANES);
    auto put = [&](uint32_t ch, const float* e) {
        if (ch >= chunks) return;
        hk_f16x8 h, l;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            // element order: pairs (k, k + 4) of what was loaded; Q8 takes the columns in order
            const float f = bad ? 0.0f : ldexpf(kind == HK_Q8 ? e[k] : e[(k >> 1) + 4 * (k & 1)], E);
            h[k] = (_Float16)f;
            if constexpr (PLANES == 2) l[k] = (_Float16)(f - (float)h[k]);
        }
        uint8_t* p = out + (size_t)(ch >> 4) * (256u * PLANES) + (ch & 15u) * 16u;
        *reinterpret_cast<hk_f16x8*>(p) = h;
        if constexpr (PLANES == 2) *reinterpret_cast<hk_f16x8*>(p + 256u) = l;
    };
#pragma unroll
    for (int i = 0; i < NC; ++i) put(me + (uint32_t)i * TPR, v[i]);
    for (uint32_t ch = me + NC * TPR; ch < chunks; ch += TPR) {
        float e[8];
        load(ch, e);
        put(ch, e);
    }
}

template <int TYPE, int PLANES>
static hipError_t image_go(const void* x, size_t stride, uint32_t n, uint32_t cols, int kind, const RowsWs& ws,
                           const int32_t* offsets, uint32_t groups, uint32_t n_pos, uint32_t tile_rows, uint32_t* status,
                           hipStream_t s) {
    const uint32_t chunks = rows_stages(kind, cols) * 16u, extra = offsets ? 1u : 0u;
    const size_t es = TYPE == HK_T_F32 ? 4 : 2;
    const bool vec = stride % 4 == 0 && reinterpret_cast<uintptr_t>(x) % (4 * es) == 0;
    // a wave a row where that holds the row in registers and fills the device
    if (chunks <= 256u && n >= 2048u)
        hipLaunchKernelGGL((rows_image_kernel<TYPE, PLANES, 64>), dim3((n + 3u) / 4u + extra), dim3(256), 0, s, x, stride, n,
                           cols, kind, chunks, vec, ws, offsets, groups, n_pos, tile_rows, status);
    else
        hipLaunchKernelGGL((rows_image_kernel<TYPE, PLANES, 256>), dim3(n + extra), dim3(256), 0, s, x, stride, n, cols, kind,
                           chunks, vec, ws, offsets, groups, n_pos, tile_rows, status);
    return hipGetLastError();
}

hipError_t launch_rows_image(const void* x, int x_type, size_t x_stride, uint32_t n, uint32_t cols, int kind, int planes,
                             const RowsWs& ws, const int32_t* offsets, uint32_t groups, uint32_t n_pos, uint32_t tile_rows,
                             uint32_t* status, hipStream_t s) {
    if (x_type == HK_T_F32)
        return planes == 2 ? image_go<HK_T_F32, 2>(x, x_stride, n, cols, kind, ws, offsets, groups, n_pos, tile_rows, status, s)
                           : image_go<HK_T_F32, 1>(x, x_stride, n, cols, kind, ws, offsets, groups, n_pos, tile_rows, status, s);
    if (x_type == HK_T_BF16)
        return image_go<HK_T_BF16, 1>(x, x_stride, n, cols, kind, ws, offsets, groups, n_pos, tile_rows, status, s);
    return image_go<HK_T_F16, 1>(x, x_stride, n, cols, kind, ws, offsets, groups, n_pos, tile_rows, status, s);
}

hipError_t launch_rows_vec_image(const void* x, int x_type, size_t x_stride, uint32_t n, uint32_t cols, int kind,
                                 const RowsWs& ws, const int32_t* offsets, uint32_t groups, uint32_t n_pos, uint32_t tile_rows,
                                 uint32_t* status, hipStream_t s) {
    switch (kind) {
    case HK_Q4: return launch_rows_vec_image_q4(x, x_type, x_stride, n, cols, ws, offsets, groups, n_pos, tile_rows, status, s);
    case HK_Q8: return launch_rows_vec_image_q8(x, x_type, x_stride, n, cols, ws, offsets, groups, n_pos, tile_rows, status, s);
    case HK_U3: return launch_rows_vec_image_u3(x, x_type, x_stride, n, cols, ws, offsets, groups, n_pos, tile_rows, status, s);
    case HK_BIN: return launch_rows_vec_image_bin(x, x_type, x_stride, n, cols, ws, offsets, groups, n_pos, tile_rows, status, s);
    case HK_MIXED: return launch_rows_vec_image_mixed(x, x_type, x_stride, n, cols, ws, offsets, groups, n_pos, tile_rows, status, s);
    }
    return hipErrorInvalidValue;
}

size_t rows_vec_image_bytes(int kind, uint32_t cols) {
    switch (kind) {
    case HK_Q4: return x_lds_bytes<HK_Q4>(n_steps_for(kind, cols));
    case HK_Q8: return x_lds_bytes<HK_Q8>(n_steps_for(kind, cols));
    case HK_U3: return x_lds_bytes<HK_U3>(n_steps_for(kind, cols));
    case HK_BIN: return x_lds_bytes<HK_BIN>(n_steps_for(kind, cols));
    default: return x_lds_bytes<HK_MIXED>(n_steps_for(kind, cols));
    }
}

hipError_t launch_rows_product(const RowsShape& sh, const RowsArgs& a, hipStream_t s) {
    switch (sh.kind) {
    case HK_Q4: return launch_rows_q4(sh, a, s);
    case HK_Q8: return launch_rows_q8(sh, a, s);
    case HK_U3: return launch_rows_u3(sh, a, s);
    case HK_BIN: return launch_rows_bin(sh, a, s);
    case HK_MIXED: return launch_rows_mixed(sh, a, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace hk
