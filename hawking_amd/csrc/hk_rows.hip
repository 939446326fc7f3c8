// hk_rows.hip -- row images and the position tiles of a product (hk_rows.h).
#include "hk_rows.h"

namespace hk {

// ------------------------------------------------------------------ row images

// Four consecutive elements of a row as f32.
template <int TYPE>
__device__ __forceinline__ void row_load4(const void* x, size_t at, bool vec, float* v) {
    if constexpr (TYPE == HK_T_F32) {
        const float* p = static_cast<const float*>(x) + at;
        if (vec) {
            const float4 f = ldg(reinterpret_cast<const float4*>(p));
            v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = ldg(p + i);
        }
    } else {
        const uint16_t* p = static_cast<const uint16_t*>(x) + at;
        uint32_t h[4];
        if (vec) {
            const uint2 w = ldg(reinterpret_cast<const uint2*>(p));
            h[0] = w.x & 0xFFFFu, h[1] = w.x >> 16, h[2] = w.y & 0xFFFFu, h[3] = w.y >> 16;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) h[i] = ldg(p + i);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v[i] = TYPE == HK_T_BF16 ? __builtin_bit_cast(float, h[i] << 16) : f16_bits_to_f32((uint16_t)h[i]);
    }
}

// The positions [first, last) of every group cut into tiles of tile_rows, in
// group order.  One block; offsets outside [0, n] or out of order are clamped,
// so whatever they hold a tile lies inside the positions.
__device__ void rows_tiles(const RowsWs& ws, const int32_t* offsets, uint32_t groups, uint32_t n, uint32_t tile_rows,
                           uint32_t* pre) {
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    __shared__ uint32_t wsum[4], lo_s[256];
    uint32_t base = 0;
    for (uint32_t g0 = 0; g0 < groups; g0 += 256u) {
        const uint32_t g = g0 + tid;
        uint32_t lo = 0, hi = 0;
        if (g < groups) {
            lo = min((uint32_t)max(offsets[g], 0), n);
            hi = max(min((uint32_t)max(offsets[g + 1], 0), n), lo);
        }
        const uint32_t c = (hi - lo + tile_rows - 1u) / tile_rows;
        const uint32_t inc = wave_incl_scan(c);
        __syncthreads();  // the last round's readers are done
        if (lane == 63u) wsum[wave] = inc;
        lo_s[tid] = lo;
        __syncthreads();
        uint32_t before = 0, total = 0;
#pragma unroll
        for (uint32_t w = 0; w < 4; ++w) {
            if (w < wave) before += wsum[w];
            total += wsum[w];
        }
        pre[tid] = before + inc - c;  // tiles of the round before this group
        __syncthreads();
        for (uint32_t j = tid; j < total; j += 256u) {
            // the last group that begins at or before tile j and has tiles: pre is ascending, empty groups share the next one's start
            uint32_t a = 0, b = 256u;
            while (b - a > 1u) {
                const uint32_t mid = (a + b) / 2u;
                if (pre[mid] <= j) a = mid; else b = mid;
            }
            const uint32_t first = lo_s[a] + (j - pre[a]) * tile_rows;
            const uint32_t end = max(min((uint32_t)max(offsets[g0 + a + 1u], 0), n), lo_s[a]);
            if (base + j < ws.max_tiles) ws.tiles[base + j] = RowsTile{g0 + a, first, min(first + tile_rows, end), 0u};
        }
        base += total;
    }
    for (uint32_t j = base + tid; j < ws.max_tiles; j += 256u) ws.tiles[j] = RowsTile{0u, 0u, 0u, 0u};  // no positions
}

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
            row_load4<TYPE>(x, base + c, vec, v);
            row_load4<TYPE>(x, base + c + apart, vec, v + 4);
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
