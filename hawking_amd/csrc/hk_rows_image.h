// hk_rows_image.h -- what the kernels that read a product's rows share: the
// element types and the cutting of the groups into position tiles.
#pragma once

#include "hk_rows.h"

namespace hk {

// Four consecutive elements of a row as f32.
__device__ __forceinline__ void row_load4(int type, const void* x, size_t at, bool vec, float* v) {
    if (type == HK_T_F32) {
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
            v[i] = type == HK_T_BF16 ? __builtin_bit_cast(float, h[i] << 16) : f16_bits_to_f32((uint16_t)h[i]);
    }
}

// The positions [first, last) of every group cut into tiles of tile_rows, in
// group order.  One block; offsets outside [0, n] or out of order are clamped,
// so whatever they hold a tile lies inside the positions.
__device__ inline void rows_tiles(const RowsWs& ws, const int32_t* offsets, uint32_t groups, uint32_t n, uint32_t tile_rows,
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

}  // namespace hk
