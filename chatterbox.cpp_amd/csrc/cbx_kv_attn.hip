// cbx_kv_attn.hip -- attention over a paged cache (cbx_kv_attend,
// include/cbx_kv.h): out = softmax(scale q K^T) V per row and query head, over
// the positions that the row sees, found through its stream's page table.
//
// A row's positions [0, n) are its prefix's [0, plen), in the prefix's pages,
// then its own, in its own pages from their first place on.  The softmax is
// taken in one pass: over any set of keys, (m, s, o) = (max x, sum e^(x - m),
// sum e^(x - m) v), and two sets' join as
//   m = max(m1, m2), s = s1 e^(m1 - m) + s2 e^(m2 - m), o alike; out = o / s,
// so keys may be cut anywhere: over lanes, waves, workgroups, and into a
// prefix's part computed once for many rows and each row's own.
//
//  * kv_rows: the step form, one row a stream, on the vector units: what
//    bounds it is reading each stream's keys and values.
//  * kv_tiles: the prompt form, and the step form's shared prefixes: 16 (row,
//    head) pairs a wave on the fp32 matrix cores.
//  * kv_join: the parts of rows whose keys were cut over workgroups.
// e^x as 2^(x log2 e): the difference x - m is formed first, so that the
// product's rounding is relative to it.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "cbx_attn_out.h"
#include "cbx_internal.h"

namespace cbx {
namespace {

constexpr int kDim = 64;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr uint32_t kNoRow = ~0u;  // a key without a page

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(__fmul_rn(d, kLog2e)); }

struct KvArgs {
    const void* kc;  // this layer's pages: [page][n_kv][position][64]
    const void* vc;
    int32_t n_pages, n_kv, shift;  // page_size = 1 << shift
    int32_t n_streams, n_prefix, max_pages;
    const int32_t* tables;
    const int32_t* parent;
    const int32_t* prefix_len;
    int32_t n_rows, n_tiles, tile_rows;
    const int32_t* row_start;
    const int32_t* position;
    const int32_t* slot;
    const int4* tiles;
    const int32_t* order;   // step form
    const float* q;
    int64_t ld_q;
    const float* k;         // the new rows, or NULL
    const float* v;
    int64_t ld_kv;
    int32_t n_head, group;  // query heads, of them per key head
    float scale;
    AttnOut o;
    // parts of rows cut over workgroups, [part][n_rows][n_head]: (m, s) and
    // o[64]; the rows' own parts first, then their prefixes' (n_own 0: none,
    // the rows are whole)
    float2* part_ms;
    float* part_o;
    int32_t n_own, n_shared;
};

// Stream i's prefix as cbx_kv_build counts it: its table's stream and the
// positions shared (0: none).
__device__ __forceinline__ int prefix_of(const KvArgs& a, int i, int& plen) {
    plen = 0;
    if (!a.parent || i < a.n_prefix || i >= a.n_streams) return -1;
    const int p = a.parent[i];
    if (p < 0 || p >= a.n_prefix) return -1;
    plen = min(max(a.prefix_len[i], 0), a.max_pages << a.shift);
    return p;
}

// The row of [page][n_kv][position] that holds place `off` of a page, head
// `kvh` (n_pages * n_kv * page_size is below 2^32).
__device__ __forceinline__ uint32_t cache_row(const KvArgs& a, int page, int kvh, int off) {
    return page < 0 || page >= a.n_pages
               ? kNoRow
               : (((uint32_t)page * (uint32_t)a.n_kv + (uint32_t)kvh) << a.shift) +
                     ((uint32_t)off & ((1u << a.shift) - 1));
}

// Dimensions [d, d + N) of a cache row, as floats.
template <class T>
__device__ __forceinline__ f4 load4(const T* base, uint32_t row, int d) {
    const T* const p = base + ((uint64_t)row << 6) + d;
    if constexpr (sizeof(T) == 4) {
        return *reinterpret_cast<const f4*>(p);
    } else {
        const h4 x = *reinterpret_cast<const h4*>(p);
        return f4{(float)x[0], (float)x[1], (float)x[2], (float)x[3]};
    }
}

// ------------------------------------------------------------------ step form

constexpr int kRowWaves = 4;
// Pages whose ids a workgroup holds at once.
constexpr int kIds = 512;
// Keys that a part of a row's own has at least (below, the row takes fewer).
constexpr int kMinPart = 64;

// One part of one row's keys, for G of its key head's query heads.  The part's
// page ids go to LDS; the waves take batches of keys in turn, LPK lanes to a
// key (16 bytes of it each), kU keys per lane in flight; each lane group keeps
// a running (m, s, o) of its keys, joined over the groups and waves in a fixed
// order.  The row's new k and v come from its input row, stored on the way.
template <class T, int G>
__global__ __launch_bounds__(64 * kRowWaves) void kv_rows(KvArgs a) {
    constexpr int DPL = 16 / sizeof(T), LPK = kDim / DPL, KPI = 64 / LPK;  // dims a lane, lanes a key
    constexpr int kU = G > 2 ? 4 : 6;
    __shared__ int32_t ids[kIds];
    __shared__ __align__(16) float new_k[kDim], new_v[kDim];
    __shared__ float red_m[kRowWaves][G], red_s[kRowWaves][G];
    __shared__ __align__(16) float red_o[kRowWaves][G][kDim];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int chunks = (a.group + G - 1) / G;
    const int r = blockIdx.x / (a.n_kv * chunks), y = blockIdx.x % (a.n_kv * chunks);
    const int kvh = y / chunks, g0 = y % chunks * G, h0 = kvh * a.group + g0;
    const int ng = min(G, a.group - g0), part = blockIdx.y;
    const int pos = a.position[r];
    int plen;
    const int pre = prefix_of(a, r, plen);
    // keys [c0, c1) of the row: its own alone where tiles take the prefix
    const int cap = a.max_pages << a.shift;
    const int lo = a.tiles ? min(plen, pos + 1) : 0;
    const int end = min(pos + 1, plen + cap);
    const int L = max(end - lo, 0), used = min(a.n_own > 0 ? a.n_own : 1, (L + kMinPart - 1) / kMinPart);
    const int size = used > 0 ? (L + used - 1) / used : 0;
    const int c0 = lo + part * size, c1 = part < used ? min(c0 + size, end) : c0;
    if (c0 >= c1) {  // no keys
        if (a.n_own > 0) {
            if (tid < ng)
                a.part_ms[((int64_t)part * a.n_rows + r) * a.n_head + h0 + tid] = float2{-INFINITY, 0.0f};
        } else if (w == 0) {
            for (int g = 0; g < ng; ++g) attn_store(a.o, r, h0 + g, lane, 0.0f);
        }
        return;
    }
    const T* const kc = static_cast<const T*>(a.kc);
    const T* const vc = static_cast<const T*>(a.vc);
    const bool has_new = a.k != nullptr && pos >= c0 && pos < c1;
    if (has_new && w == 0) {
        // rounded as the cache holds it
        const T kn = (T)a.k[r * a.ld_kv + kvh * kDim + lane];
        const T vn = (T)a.v[r * a.ld_kv + kvh * kDim + lane];
        new_k[lane] = (float)kn;
        new_v[lane] = (float)vn;
        const int s = a.slot[r];
        const uint32_t row = cache_row(a, s < 0 ? -1 : s >> a.shift, kvh, s);
        if (g0 == 0 && row != kNoRow) {
            const_cast<T*>(kc)[((uint64_t)row << 6) + lane] = kn;
            const_cast<T*>(vc)[((uint64_t)row << 6) + lane] = vn;
        }
    }
    // whether the new position is one that the row sees
    const bool new_ok = has_new && a.slot[r] >= 0 && (a.slot[r] >> a.shift) < a.n_pages;
    const int sub = lane / LPK, d0 = lane % LPK * DPL;
    float q[G][DPL], o[G][DPL], m[G], s[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const float* const qr = a.q + r * a.ld_q + (h0 + min(g, ng - 1)) * kDim + d0;
#pragma unroll
        for (int d = 0; d < DPL; d += 4) {
            const f4 x = *reinterpret_cast<const f4*>(qr + d);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                q[g][d + e] = __fmul_rn(x[e], a.scale);
                o[g][d + e] = 0.0f;
            }
        }
        m[g] = -INFINITY;
        s[g] = 0.0f;
    }
    const int32_t* const own_t = a.tables + (int64_t)r * a.max_pages;
    const int32_t* const pre_t = a.tables + (int64_t)max(pre, 0) * a.max_pages;
    const int ps = 1 << a.shift;
    for (int s0 = c0; s0 < c1;) {
        // the ids of [s0, s1): the prefix's pages, then the row's own
        const int in_pre = s0 < plen ? ((min(c1, plen) - 1) >> a.shift) - (s0 >> a.shift) + 1 : 0;
        const int n_pre = min(in_pre, kIds);
        const int a0 = s0 >> a.shift, b0 = (max(s0, plen) - plen) >> a.shift;
        int s1 = n_pre < in_pre || plen >= c1 ? min(c1, (a0 + n_pre) << a.shift)
                                               : min((int64_t)c1, plen + (((int64_t)b0 + kIds - n_pre) << a.shift));
        if (plen >= c1) s1 = min(s1, c1);
        const int n_own_pages = s1 > plen ? ((s1 - 1 - plen) >> a.shift) - b0 + 1 : 0;
        if (s0 != c0) __syncthreads();
        for (int i = tid; i < n_pre + n_own_pages; i += 64 * kRowWaves)
            ids[i] = i < n_pre ? pre_t[a0 + i] : own_t[b0 + i - n_pre];
        __syncthreads();
        for (int j0 = s0 + w * KPI * kU; j0 < s1; j0 += kRowWaves * KPI * kU) {
            float kk[kU][DPL], vv[kU][DPL], x[kU][G];
            bool on[kU];
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const int j = min(j0 + KPI * u + sub, s1 - 1);
                const bool theirs = j < plen;
                const int place = theirs ? j : j - plen;
                const int id = ids[(place >> a.shift) - (theirs ? a0 : b0 - n_pre)];
                const uint32_t row = cache_row(a, id, kvh, place & (ps - 1));
                on[u] = j0 + KPI * u + sub < s1 && (has_new && j == pos ? new_ok : row != kNoRow);
                const uint32_t at = row == kNoRow ? 0 : row;
#pragma unroll
                for (int d = 0; d < DPL; d += 4) {
                    const f4 kx = load4(kc, at, d0 + d), vx = load4(vc, at, d0 + d);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        kk[u][d + e] = kx[e];
                        vv[u][d + e] = vx[e];
                    }
                }
            }
            if (has_new && pos >= j0 && pos < j0 + KPI * kU) {
#pragma unroll
                for (int u = 0; u < kU; ++u)
                    if (j0 + KPI * u + sub == pos) {
#pragma unroll
                        for (int d = 0; d < DPL; ++d) {
                            kk[u][d] = new_k[d0 + d];
                            vv[u][d] = new_v[d0 + d];
                        }
                    }
            }
#pragma unroll
            for (int g = 0; g < G; ++g) {
                float bm = m[g];
#pragma unroll
                for (int u = 0; u < kU; ++u) {
                    float t = 0.0f;
#pragma unroll
                    for (int d = 0; d < DPL; ++d) t = __fmaf_rn(q[g][d], kk[u][d], t);
                    t = __fadd_rn(t, dpp16<0xB1>(t));   // the key's lanes
                    t = __fadd_rn(t, dpp16<0x4E>(t));
                    t = __fadd_rn(t, dpp16<0x141>(t));
                    if (LPK == 16) t = __fadd_rn(t, dpp16<0x140>(t));
                    x[u][g] = t;
                    if (on[u]) bm = fmaxf(bm, t);
                }
                if (bm > m[g]) {
                    const float f = exp_of(__fsub_rn(m[g], bm));  // 0 from -inf
                    s[g] = __fmul_rn(s[g], f);
#pragma unroll
                    for (int d = 0; d < DPL; ++d) o[g][d] = __fmul_rn(o[g][d], f);
                    m[g] = bm;
                }
#pragma unroll
                for (int u = 0; u < kU; ++u) {
                    // a key that is -inf while no other is larger has no weight
                    if (on[u] && !(x[u][g] == -INFINITY)) {
                        const float e = exp_of(__fsub_rn(x[u][g], m[g]));
                        s[g] = __fadd_rn(s[g], e);
#pragma unroll
                        for (int d = 0; d < DPL; ++d) o[g][d] = __fmaf_rn(e, vv[u][d], o[g][d]);
                    }
                }
            }
        }
        s0 = s1;
    }
    // the groups of a wave, then the waves, joined in order
#pragma unroll
    for (int g = 0; g < G; ++g) {
#pragma unroll
        for (int x = LPK; x < 64; x <<= 1) {
            const float mo = __shfl_xor(m[g], x), so = __shfl_xor(s[g], x);
            const float M = fmaxf(m[g], mo);
            const float f = m[g] == -INFINITY ? 0.0f : exp_of(__fsub_rn(m[g], M));
            const float fo = mo == -INFINITY ? 0.0f : exp_of(__fsub_rn(mo, M));
            s[g] = __fadd_rn(__fmul_rn(s[g], f), __fmul_rn(so, fo));
#pragma unroll
            for (int d = 0; d < DPL; ++d)
                o[g][d] = __fadd_rn(__fmul_rn(o[g][d], f), __fmul_rn(__shfl_xor(o[g][d], x), fo));
            m[g] = M;
        }
        if (lane == 0) {
            red_m[w][g] = m[g];
            red_s[w][g] = s[g];
        }
        if (sub == 0) {
#pragma unroll
            for (int d = 0; d < DPL; ++d) red_o[w][g][d0 + d] = o[g][d];
        }
    }
    __syncthreads();
    for (int g = w; g < ng; g += kRowWaves) {
        float M = red_m[0][g];
#pragma unroll
        for (int i = 1; i < kRowWaves; ++i) M = fmaxf(M, red_m[i][g]);
        float st = 0.0f, ot = 0.0f;
#pragma unroll
        for (int i = 0; i < kRowWaves; ++i) {
            const float f = red_m[i][g] == -INFINITY ? 0.0f : exp_of(__fsub_rn(red_m[i][g], M));
            st = __fadd_rn(st, __fmul_rn(red_s[i][g], f));
            ot = __fadd_rn(ot, __fmul_rn(red_o[i][g][lane], f));
        }
        if (a.n_own > 0) {
            const int64_t at = ((int64_t)part * a.n_rows + r) * a.n_head + h0 + g;
            if (lane == 0) a.part_ms[at] = float2{M, st};
            a.part_o[at * kDim + lane] = ot;
        } else {
            attn_store(a.o, r, h0 + g, lane, st == 0.0f ? 0.0f : __fdiv_rn(ot, st));
        }
    }
}

// ------------------------------------------------------------------ joins

// One wave per row and head: the row's own parts and its prefix's.
__global__ __launch_bounds__(256) void kv_join(KvArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t x = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (x >= (int64_t)a.n_rows * a.n_head) return;
    const int r = (int)(x / a.n_head), h = (int)(x % a.n_head);
    const int64_t rows = (int64_t)a.n_rows * a.n_head;
    int plen;
    prefix_of(a, r, plen);
    // parts of this row: none without a position
    const bool live = a.position[r] >= 0;
    const int n = live ? a.n_own + (plen > 0 ? a.n_shared : 0) : 0;
    float M = -INFINITY, st = 0.0f, ot = 0.0f;
    for (int p0 = 0; p0 < n; p0 += 64) {
        const float2 ms = p0 + lane < n ? a.part_ms[(p0 + lane) * rows + x] : float2{-INFINITY, 0.0f};
        float bm = ms.x;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) bm = fmaxf(bm, __shfl_xor(bm, o));
        const float nm = fmaxf(M, bm);
        const float keep = M == -INFINITY ? 0.0f : exp_of(__fsub_rn(M, nm));
        st = __fmul_rn(st, keep);
        ot = __fmul_rn(ot, keep);
        M = nm;
        const float f = ms.x == -INFINITY ? 0.0f : exp_of(__fsub_rn(ms.x, M));
        const float sf = __fmul_rn(ms.y, f);
        for (uint64_t left = __ballot(!(ms.y == 0.0f)); left; left &= left - 1) {
            const int i = (int)__builtin_ctzll(left);
            st = __fadd_rn(st, __shfl(sf, i));
            ot = __fadd_rn(ot, __fmul_rn(__shfl(f, i), a.part_o[((p0 + i) * rows + x) * kDim + lane]));
        }
    }
    attn_store(a.o, r, h, lane, st == 0.0f ? 0.0f : __fdiv_rn(ot, st));
}

// ------------------------------------------------------------------ tiles

// The prompt form's new rows to their slots, before any row attends.
template <class T>
__global__ __launch_bounds__(256) void kv_store(KvArgs a) {
    const int r = blockIdx.x, s = a.slot[r];
    if (s < 0 || (s >> a.shift) >= a.n_pages) return;
    for (int i = threadIdx.x; i < a.n_kv * 16; i += 256) {
        const int kvh = i >> 4, d = 4 * (i & 15);
        const uint64_t at = ((uint64_t)cache_row(a, s >> a.shift, kvh, s) << 6) + d;
        const f4 k = *reinterpret_cast<const f4*>(a.k + r * a.ld_kv + kvh * kDim + d);
        const f4 v = *reinterpret_cast<const f4*>(a.v + r * a.ld_kv + kvh * kDim + d);
        T* const kc = static_cast<T*>(const_cast<void*>(a.kc)) + at;
        T* const vc = static_cast<T*>(const_cast<void*>(a.vc)) + at;
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<f4*>(kc) = k;
            *reinterpret_cast<f4*>(vc) = v;
        } else {
            *reinterpret_cast<h4*>(kc) = h4{(T)k[0], (T)k[1], (T)k[2], (T)k[3]};
            *reinterpret_cast<h4*>(vc) = h4{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
        }
    }
}

__device__ __forceinline__ f4 mfma_f32(float x, float y, const f4& acc) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(x, y, acc, 0, 0, 0);
}

// A wave takes 16 (row, head) pairs of a tile and one key head and walks its
// keys 32 at a time with v_mfma_f32_16x16x4_f32.
//  * Scores transposed, S^T = K Q^T: lane (g = l / 16, c = l % 16) feeds key c
//    and pair c at dimensions 16 cc + 4 g + e (step (cc, e)), and holds pair
//    c's scores at keys 4 g + v: its own pair's limit, maximum and sum, joined
//    over g by two exchanges.
//  * P V: those exponentials are the A operand as they stand (pair c, step v:
//    key 4 g + v), V[4 g + v][4 c ..] the B operand, one 16-byte load for four
//    output tiles, so lane (g, c) ends with pairs 4 g + v at dimensions
//    4 c .. 4 c + 3.
// A key that a pair does not see has weight 0, and 0 times a V that is not
// finite would reach the pair: where some pair does not see all 32 keys, such
// values are looked for, and if there are any, added pair by pair with the
// unseen keys' V at 0.
// KS = 4: the workgroup's four waves take the same pairs and every fourth
// 32 keys, joined through LDS; KS = 1: each wave its own pairs.
// PART: the step form's prefixes: keys cut over blockIdx.y, parts stored.
template <class T, int KS, bool PART>
__global__ __launch_bounds__(256) void kv_tiles(KvArgs a) {
    constexpr int KT = 2;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int g = lane >> 4, c = lane & 15;
    const int kvh = blockIdx.x % a.n_kv, unit = blockIdx.x / a.n_kv;
    const T* const kc = static_cast<const T*>(a.kc);
    const T* const vc = static_cast<const T*>(a.vc);
    if (!PART) {  // rows behind the last
        const int total = a.row_start[a.n_streams];
        for (int64_t r = (int64_t)max(total, 0) + blockIdx.x; r < a.n_rows; r += gridDim.x)
            for (int h = w; h < a.n_head; h += 4) attn_store(a.o, (int)r, h, lane, 0.0f);
    }
    const int4 tile = a.tiles[KS == 1 ? unit : unit / 4];
    const int p = 16 * (KS == 1 ? w : unit % 4) + c;
    const int count = min(tile.z, a.tile_rows);
    const int first = min(max(tile.y, 0), a.n_rows);
    const int at = first + p / a.group, h = kvh * a.group + p % a.group;
    bool real = tile.x >= 0 && tile.x < a.n_streams && p < count * a.group && at < a.n_rows;
    int row = -1;
    if (real) row = PART ? a.order[at] : at;
    real = real && row >= 0 && row < a.n_rows;
    if (!__ballot(real)) return;  // a whole workgroup, or no barrier follows
    const int rc = real ? row : 0;
    // lim: the last key the pair sees
    int plen = 0, pre = -1, lim;
    if (PART) {
        prefix_of(a, rc, lim);
        lim = real ? lim - 1 : -1;
    } else {
        pre = prefix_of(a, tile.x, plen);
        lim = real ? min(a.position[rc], plen + (a.max_pages << a.shift) - 1) : -1;
    }
    int last = lim, least = real ? lim : INT32_MAX;
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) {
        last = max(last, __shfl_xor(last, x));
        least = min(least, __shfl_xor(least, x));
    }
    last = __builtin_amdgcn_readfirstlane(last);
    least = __builtin_amdgcn_readfirstlane(least);
    int begin = 0, end = last + 1;
    if (PART) {  // this workgroup's keys, the same for all pairs of the tile
        const int keys = min(max(tile.w, 0), a.max_pages << a.shift);
        const int used = min(a.n_shared, (keys + kMinPart - 1) / kMinPart);
        const int size = used > 0 ? ((keys + used - 1) / used + 15) / 16 * 16 : 0;
        begin = min((int)blockIdx.y * size, keys);
        end = min(end, min(begin + size, keys));
    }
    f4 q[4], o[4];
    {
        const float* const qr = a.q + rc * a.ld_q + (real ? h : 0) * kDim + 4 * g;
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) {
            q[cc] = *reinterpret_cast<const f4*>(qr + 16 * cc) * a.scale;
            o[cc] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    const int32_t* const own_t = a.tables + (int64_t)min(max(tile.x, 0), a.n_streams - 1) * a.max_pages;
    const int32_t* const pre_t = a.tables + (int64_t)max(pre, 0) * a.max_pages;
    float m = -INFINITY, s = 0.0f;
    for (int j0 = begin + (KS == 1 ? 0 : 16 * KT * w); j0 < end; j0 += 16 * KT * KS) {
        // lane l: where key j0 + l % 32 is (keys past the end: the last's)
        const int jl = min(j0 + (lane & 31), end - 1);
        const bool theirs = jl < plen;
        const int place = theirs ? jl : jl - plen;
        const uint32_t where =
            cache_row(a, (theirs ? pre_t : own_t)[place >> a.shift], kvh, place);
        // the keys with a page, a bit each
        const uint32_t paged = (uint32_t)__ballot(where != kNoRow);
        f4 kk[KT][4], vv[KT][4], x[KT];
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
            uint32_t kr = (uint32_t)__shfl((int)where, 16 * kt + c);
            kr = kr == kNoRow ? 0 : kr;
#pragma unroll
            for (int cc = 0; cc < 4; ++cc) kk[kt][cc] = load4(kc, kr, 16 * cc + 4 * g);
        }
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                uint32_t vr = (uint32_t)__shfl((int)where, 16 * kt + 4 * g + v);
                const bool none = vr == kNoRow;
                vv[kt][v] = load4(vc, none ? 0 : vr, 4 * c);
                if (none) vv[kt][v] = f4{0.0f, 0.0f, 0.0f, 0.0f};
            }
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) x[kt] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int cc = 0; cc < 4; ++cc)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) x[kt] = mfma_f32(kk[kt][cc][e], q[cc][e], x[kt]);
        const auto seen = [&](int kt, int v) {
            const int k = 16 * kt + 4 * g + v;
            return j0 + k <= lim && j0 + k < end && (paged >> k & 1);
        };
        float bm = -INFINITY;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int v = 0; v < 4; ++v)
                if (seen(kt, v)) bm = fmaxf(bm, x[kt][v]);
        bm = fmaxf(bm, __shfl_xor(bm, 16));
        bm = fmaxf(bm, __shfl_xor(bm, 32));
        if (__ballot(bm > m)) {
            const float nm = fmaxf(m, bm);
            const float f = m == -INFINITY ? 0.0f : exp_of(__fsub_rn(m, nm));
            s = __fmul_rn(s, f);
            m = nm;
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const float fv = __shfl(f, 4 * g + v);  // pair 4 g + v's
#pragma unroll
                for (int dt = 0; dt < 4; ++dt) o[dt][v] = __fmul_rn(o[dt][v], fv);
            }
        }
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const bool on = seen(kt, v) && !(x[kt][v] == -INFINITY);
                x[kt][v] = on ? exp_of(__fsub_rn(x[kt][v], m)) : 0.0f;
                s = __fadd_rn(s, x[kt][v]);
            }
        bool plain = true;
        if (j0 + 16 * KT - 1 > least || j0 + 16 * KT > end) {
            float z = 0.0f;  // NaN once a value is not finite
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int v = 0; v < 4; ++v)
#pragma unroll
                    for (int dt = 0; dt < 4; ++dt) z = __fmaf_rn(vv[kt][v][dt], 0.0f, z);
            plain = __ballot(z != z) == 0;
        }
        if (plain) {
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int v = 0; v < 4; ++v)
#pragma unroll
                    for (int dt = 0; dt < 4; ++dt) o[dt] = mfma_f32(x[kt][v], vv[kt][v][dt], o[dt]);
        } else {
#pragma unroll 1
            for (int i = 0; i < 16; ++i) {
                const int li = __builtin_amdgcn_readlane(lim, i);
#pragma unroll
                for (int dt = 0; dt < 4; ++dt) {
                    f4 add = o[dt];
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                        for (int v = 0; v < 4; ++v) {
                            const int j = j0 + 16 * kt + 4 * g + v;
                            add = mfma_f32(x[kt][v], j <= li && j < end ? vv[kt][v][dt] : 0.0f, add);
                        }
#pragma unroll
                    for (int v = 0; v < 4; ++v)
                        if (4 * g + v == i) o[dt][v] = add[v];
                }
            }
        }
    }
    s = __fadd_rn(s, __shfl_xor(s, 16));  // the pair's sum over its four lanes
    s = __fadd_rn(s, __shfl_xor(s, 32));
    // pair i's (m, s, o): a part, or the row's outputs
    const auto store = [&](int i, float pm, float psum, const f4& po) {
        const int ri = __shfl(real ? row : a.n_rows, i), hi = __shfl(h, i);
        if (PART) {
            if (ri >= a.n_rows) return;
            const int64_t to = ((int64_t)(a.n_own + blockIdx.y) * a.n_rows + ri) * a.n_head + hi;
            if (c == 0) a.part_ms[to] = float2{pm, psum};
            *reinterpret_cast<f4*>(a.part_o + to * kDim + 4 * c) = po;
        } else {
            f4 y;
#pragma unroll
            for (int dt = 0; dt < 4; ++dt) y[dt] = psum == 0.0f ? 0.0f : __fdiv_rn(po[dt], psum);
            attn_store4(a.o, a.n_rows, ri, hi, c, y);
        }
    };
    if constexpr (KS == 1) {
#pragma unroll
        for (int v = 0; v < 4; ++v)
            store(4 * g + v, __shfl(m, 4 * g + v), __shfl(s, 4 * g + v),
                  f4{o[0][v], o[1][v], o[2][v], o[3][v]});
    } else {
        // wave w joins the four waves' pairs 4 g + w
        __shared__ f4 os[KS][4][64];
        __shared__ float ms[KS][16], ss[KS][16];
#pragma unroll
        for (int v = 0; v < 4; ++v) os[w][v][lane] = f4{o[0][v], o[1][v], o[2][v], o[3][v]};
        if (g == 0) {
            ms[w][c] = m;
            ss[w][c] = s;
        }
        __syncthreads();
        const int i = 4 * g + w;
        float M = ms[0][i];
#pragma unroll
        for (int x = 1; x < KS; ++x) M = fmaxf(M, ms[x][i]);
        float st = 0.0f;
        f4 ot = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int x = 0; x < KS; ++x) {
            const float f = ms[x][i] == -INFINITY ? 0.0f : exp_of(__fsub_rn(ms[x][i], M));
            st = __fadd_rn(st, __fmul_rn(ss[x][i], f));
            const f4 ov = os[x][w][lane];
#pragma unroll
            for (int dt = 0; dt < 4; ++dt) ot[dt] = __fadd_rn(ot[dt], __fmul_rn(ov[dt], f));
        }
        store(i, M, st, ot);
    }
}

// ------------------------------------------------------------------ launches

// How a call's keys are cut: parts of a row's own (0: whole rows, stored by
// the workgroup itself) and of a prefix.
struct Cut {
    int own, shared;
};

int head_chunk(int group) { return group >= 3 ? 4 : group; }

Cut cut_of(const cbx_kv_attn& a) {
    Cut c{0, 0};
    if (a.rows->stream) return c;
    const int group = a.n_head / a.cache->n_head;
    const int chunks = (group + head_chunk(group) - 1) / head_chunk(group);
    const int64_t wgs = (int64_t)a.rows->n_rows * a.cache->n_head * chunks;
    const int64_t cap = (int64_t)a.streams->max_pages * a.cache->page_size;
    const bool tiles = a.rows->tiles && a.streams->parent && a.streams->n_prefix > 0;
    const int64_t longest = tiles || !a.streams->parent ? cap : 2 * cap;
    int64_t own = (1024 + wgs - 1) / wgs;
    own = std::max(own, (longest + 1023) / 1024);
    own = std::min(own, std::min<int64_t>(64, (longest + kMinPart - 1) / kMinPart));
    if (tiles) {
        const int64_t t = (int64_t)a.rows->n_tiles * a.cache->n_head;
        const int64_t most = std::min<int64_t>(32, (cap + kMinPart - 1) / kMinPart);
        c.shared = (int)std::min(std::max<int64_t>((1024 + t - 1) / t, 1), most);
        c.own = (int)own;
    } else {
        c.own = own > 1 ? (int)own : 0;
    }
    return c;
}

template <class T>
hipError_t launch_rows(const KvArgs& a, hipStream_t st) {
    const int G = head_chunk(a.group), chunks = (a.group + G - 1) / G;
    const dim3 grid((unsigned)a.n_rows * a.n_kv * chunks, (unsigned)max(a.n_own, 1));
    const auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(64 * kRowWaves), 0, st, a);
        return hipGetLastError();
    };
    return G == 1 ? go(kv_rows<T, 1>) : G == 2 ? go(kv_rows<T, 2>) : go(kv_rows<T, 4>);
}

template <class T>
hipError_t launch_tiles(const KvArgs& a, bool part, hipStream_t st) {
    const int64_t waves = (int64_t)a.n_tiles * 4 * a.n_kv * (part ? a.n_shared : 1);
    const bool split = waves < 2048;
    const dim3 grid((unsigned)a.n_kv * a.n_tiles * (split ? 4 : 1),
                    (unsigned)(part ? a.n_shared : 1));
    const auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, a);
        return hipGetLastError();
    };
    if (part) return split ? go(kv_tiles<T, 4, true>) : go(kv_tiles<T, 1, true>);
    return split ? go(kv_tiles<T, 4, false>) : go(kv_tiles<T, 1, false>);
}

template <class T>
hipError_t launch(const KvArgs& a, bool step, hipStream_t st) {
    hipError_t e;
    if (!step) {
        if (a.k) {
            hipLaunchKernelGGL(kv_store<T>, dim3((unsigned)a.n_rows), dim3(256), 0, st, a);
            if ((e = hipGetLastError()) != hipSuccess) return e;
        }
        return launch_tiles<T>(a, false, st);
    }
    if (a.n_shared && (e = launch_tiles<T>(a, true, st)) != hipSuccess) return e;
    if ((e = launch_rows<T>(a, st)) != hipSuccess || !a.n_own) return e;
    const int64_t waves = (int64_t)a.n_rows * a.n_head;
    hipLaunchKernelGGL(kv_join, dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace

uint64_t kv_workspace_bytes(const cbx_kv_attn& a) {
    const Cut c = cut_of(a);
    const uint64_t parts = (uint64_t)(c.own + c.shared) * a.rows->n_rows * a.n_head;
    return (parts * 8 + 255) / 256 * 256 + parts * kDim * 4;
}

hipError_t launch_kv_attend(const cbx_kv_attn& c, uint32_t* parts, float* inv, hipStream_t st) {
    const cbx_kv_cache& p = *c.cache;
    const cbx_kv_streams& s = *c.streams;
    const cbx_kv_rows& r = *c.rows;
    const Cut cut = cut_of(c);
    const size_t layer = (size_t)p.n_pages * p.n_head * p.page_size * kDim * (p.type == CBX_KV_F32 ? 4 : 2);
    KvArgs a{};
    a.kc = static_cast<const char*>(p.k) + layer * c.layer;
    a.vc = static_cast<const char*>(p.v) + layer * c.layer;
    a.n_pages = p.n_pages;
    a.n_kv = p.n_head;
    a.shift = __builtin_ctz((unsigned)p.page_size);
    a.n_streams = s.n_streams;
    a.n_prefix = s.n_prefix;
    a.max_pages = s.max_pages;
    a.tables = s.tables;
    a.parent = s.parent;
    a.prefix_len = s.prefix_len;
    a.n_rows = r.n_rows;
    a.n_tiles = r.n_tiles;
    a.tile_rows = r.tile_rows;
    a.row_start = r.row_start;
    a.position = r.position;
    a.slot = r.slot;
    // a step's tiles where streams can have prefixes
    a.tiles = r.stream || cut.shared ? reinterpret_cast<const int4*>(r.tiles) : nullptr;
    a.order = r.order;
    a.q = c.q;
    a.ld_q = c.ld_q;
    a.k = c.k;
    a.v = c.v;
    a.ld_kv = c.ld_kv;
    a.n_head = c.n_head;
    a.group = c.n_head / p.n_head;
    a.scale = c.scale;
    a.o = AttnOut{c.out, c.ld_out, parts, inv, c.n_head};
    const uint64_t n = (uint64_t)(cut.own + cut.shared) * r.n_rows * c.n_head;
    a.part_ms = static_cast<float2*>(c.workspace);
    a.part_o = reinterpret_cast<float*>(static_cast<char*>(c.workspace) + (n * 8 + 255) / 256 * 256);
    a.n_own = cut.own;
    a.n_shared = cut.shared;
    return p.type == CBX_KV_F32 ? launch<float>(a, !r.stream, st) : launch<_Float16>(a, !r.stream, st);
}

}  // namespace cbx
