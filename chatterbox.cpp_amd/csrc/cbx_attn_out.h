// cbx_attn_out.h -- where an attention kernel's output rows go: plain fp32
// rows, or split into fp16 parts for the product that reads them (cbx_split.h).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "cbx_split.h"
#include "cbx_weights.h"

namespace cbx {

struct AttnOut {
    float* out;       // [n_rows][ld]
    int64_t ld;
    uint32_t* parts;  // when set, the rows go there instead, split for the next
    float* inv;       //   product, the scales here (rows of n_head * 64)
    int32_t n_head;
};

// Element `lane` (0..63) of head h of row r's attention output, o, from one
// wave: to out, or split (the head's 64 values are blocks 2h and 2h + 1 of the
// row: lanes 0-31 and 32-63, each block scaled by its own largest magnitude,
// pairs of lanes joining their fp16 halves into dwords).
__device__ __forceinline__ void attn_store(const AttnOut& a, int r, int h, int lane, float o) {
    if (!a.parts) {
        a.out[(int64_t)r * a.ld + h * 64 + lane] = o;
        return;
    }
    float mx = fabsf(o);
#pragma unroll
    for (int q = 1; q < 32; q <<= 1) mx = fmaxf(mx, __shfl_xor(mx, q));
    float sc, sinv;
    split_scale(mx, sc, sinv);
    const float y = __fmul_rn(o, sc);
    const _Float16 hh = (_Float16)y;
    const _Float16 ll = (_Float16)__fsub_rn(y, (float)hh);
    const uint32_t hv = __builtin_bit_cast(uint16_t, hh), lv = __builtin_bit_cast(uint16_t, ll);
    const uint32_t ho = (uint32_t)__shfl_xor((int)hv, 1), lo = (uint32_t)__shfl_xor((int)lv, 1);
    const int nball = a.n_head * 2, kb = 2 * h + (lane >> 5), k = lane & 31;
    const int T = r >> 4, m = r & 15;
    if ((lane & 1) == 0) {
        // dword (k % 8) / 2 of lane 16 (k / 8) + m's hi (lo) 16 bytes
        uint32_t* const base =
            a.parts + ((int64_t)T * nball + kb) * 512 + 4 * (16 * (k >> 3) + m) + (k & 7) / 2;
        base[0] = hv | (ho << 16);
        base[256] = lv | (lo << 16);
    }
    if (k == 0) a.inv[split_inv_index(T, m, nball, kb)] = sinv;
}

// Dimensions 4c .. 4c + 3 of head h of row r's attention output from lane c
// of a 16-lane row (every lane of the wave takes part; nothing stored past
// n_rows): to out, or split as attn_store does (block 2h + c / 8, its largest
// magnitude over 8 lanes).
__device__ __forceinline__ void attn_store4(const AttnOut& a, int n_rows, int r, int h, int c,
                                            const f4& o) {
    if (!a.parts) {
        if (r < n_rows) *reinterpret_cast<f4*>(a.out + (int64_t)r * a.ld + h * 64 + 4 * c) = o;
        return;
    }
    float mx = fmaxf(fmaxf(fabsf(o[0]), fabsf(o[1])), fmaxf(fabsf(o[2]), fabsf(o[3])));
#pragma unroll
    for (int x = 1; x < 8; x <<= 1) mx = fmaxf(mx, __shfl_xor(mx, x));
    if (r >= n_rows) return;
    float sc, sinv;
    split_scale(mx, sc, sinv);
    uint32_t hi[2], lo[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float y0 = __fmul_rn(o[2 * i], sc), y1 = __fmul_rn(o[2 * i + 1], sc);
        const _Float16 h0 = (_Float16)y0, h1 = (_Float16)y1;
        hi[i] = __builtin_bit_cast(uint32_t, split_h2{h0, h1});
        lo[i] = __builtin_bit_cast(uint32_t, split_h2{(_Float16)__fsub_rn(y0, (float)h0),
                                                      (_Float16)__fsub_rn(y1, (float)h1)});
    }
    const int nball = a.n_head * 2, kb = 2 * h + (c >> 3), T = r >> 4, m = r & 15;
    // values 4 (c % 8) .. of the block: half (c & 1) of group (c % 8) / 2
    uint32_t* const d =
        a.parts + ((int64_t)T * nball + kb) * 512 + 4 * (16 * ((c & 7) >> 1) + m) + 2 * (c & 1);
    *reinterpret_cast<uint2*>(d) = make_uint2(hi[0], hi[1]);
    *reinterpret_cast<uint2*>(d + 256) = make_uint2(lo[0], lo[1]);
    if ((c & 7) == 0) a.inv[split_inv_index(T, m, nball, kb)] = sinv;
}

}  // namespace cbx
