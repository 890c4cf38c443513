// cbx_kv_attn.hip -- attention over a paged cache (cbx_kv_attend,
// include/cbx_kv.h): out = softmax(scale q K^T) V per row and query head, over
// the positions that the row sees, found through its stream's page table.
//
// A row's positions [0, n) are its prefix's [0, plen), in the prefix's pages,
// then its own, in its own pages from their first place on.  The softmax is
// taken in one pass, e^x as 2^y, y = x log2 e (the scale that queries are
// multiplied by holds log2 e): over any set of keys, with a whole number r near
// the largest y, (r, s, o) = (r, sum w, sum w v), w = 2^(y - r), and two sets join as
//   r = max(r1, r2), s = s1 2^(r1 - r) + s2 2^(r2 - r), o alike; out = o / s,
// so keys may be cut anywhere: over lanes, waves, workgroups, and into a
// prefix's part computed once for many rows and each row's own.  r whole: every
// rescaling is by a power of two.  y is one value for a key wherever it is met and
// y - r is exact where it matters (the two are near), so r leaves no rounding of its
// own, at any size of the scores.
//
//  * kv_rows: the step form, one row a stream, on the vector units: what
//    bounds it is reading each stream's keys and values.
//  * kv_tiles: the prompt form, and steps whose query heads share a key head:
//    16 (row, head) pairs a wave on the 16-bit matrix cores.
//  * kv_shared: steps with shared prefixes, a prefix's keys as tiles for all of
//    its rows, the rows' own as in kv_rows or kv_tiles.
//  * kv_join: the parts of rows whose keys were cut over workgroups.
// Times are of the kernels on an MI355X, where a large copy moves 4.77 TB/s and
// a large bf16 product runs at 1.15 PFLOP/s; 16 heads of 64 where not said.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "cbx_attn_out.h"
#include "cbx_internal.h"

namespace cbx {
namespace {

constexpr int kDim = 64;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr uint32_t kNoRow = ~0u;  // a key without a page

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));

// 2^(from - to) for references: 0 from a set without keys (-inf).
__device__ __forceinline__ float rescale(float from, float to) {
    return from == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(__fsub_rn(from, to));
}

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
    uint32_t over_group;    // x / group = x * over_group >> 16 for x < 128
    float scale;            // times log2 e
    AttnOut o;
    // parts of rows cut over workgroups, [part][n_rows][n_head]: (m, s) and
    // o[64]; the rows' own parts first, then their prefixes' (n_own 0: none,
    // the rows are whole)
    float2* part_ms;
    float* part_o;
    int32_t n_own, n_shared;
    int32_t min_part;  // keys that a part of a row's own has at least, where there are more
};

__device__ __forceinline__ int over_group(const KvArgs& a, int x) {
    return (int)((uint32_t)x * a.over_group >> 16);
}

// Stream i's prefix as cbx_kv_build counts it: its table's stream and the
// positions shared (0: none).
__device__ __forceinline__ int prefix_of(const KvArgs& a, int i, int& plen) {
    plen = 0;
    if (!a.parent || i < a.n_prefix || i >= a.n_streams) return -1;
    const int p = a.parent[i], n = a.prefix_len[i];  // both loads before the first use
    if (p < 0 || p >= a.n_prefix) return -1;
    plen = min(max(n, 0), a.max_pages << a.shift);
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

template <class T>
__device__ __forceinline__ void store4(T* base, uint32_t row, int d, const f4& x) {
    T* const p = base + ((uint64_t)row << 6) + d;
    if constexpr (sizeof(T) == 4) *reinterpret_cast<f4*>(p) = x;
    else *reinterpret_cast<h4*>(p) = h4{(T)x[0], (T)x[1], (T)x[2], (T)x[3]};
}

// ------------------------------------------------------------------ step form

// Keys that a part has at least, where there are more.
constexpr int kMinPart = 64;

// Sixteen bytes of a cache row as they are, and their values.
template <class T>
struct Chunk;
template <>
struct Chunk<float> {
    static constexpr int kN = 4;
    typedef f4 Raw;
    __device__ static __forceinline__ float at(const Raw& x, int i) { return x[i]; }
};
template <>
struct Chunk<_Float16> {
    static constexpr int kN = 8;
    typedef h8 Raw;
    __device__ static __forceinline__ float at(const Raw& x, int i) { return (float)x[i]; }
};

// One part of one row's keys, for G of its key head's query heads, by W waves
// (4: a workgroup; 1: the workgroup's waves take a head each, with no barrier).
// Bound by the bytes: 64 rows of 129 to 383 fp32 keys 29 us, 4.65 TB/s; fp16 14.8.
// LPK lanes to a key, 16 bytes of it each, kU keys per lane in flight; the page
// ids of 64 pages are held by the wave's lanes, and handed over by an exchange.
// Each lane group keeps a running (m, s, o) of its keys, joined over the groups
// and waves in a fixed order.  The row's new k and v come from its input row,
// stored on the way.
template <class T, int G, int W>
__device__ __forceinline__ void rows_of(const KvArgs& a, uint32_t block, int part) {
    using C = Chunk<T>;
    constexpr int DPL = C::kN, LPK = kDim / DPL, KPI = 64 / LPK;  // dims a lane, lanes a key
    constexpr int kU = G > 2 || sizeof(T) == 2 ? 4 : 6;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int chunks = (a.group + G - 1) / G, per_row = a.n_kv * chunks;
    const int64_t unit = W == 4 ? block : (int64_t)block * 4 + w;
    if (unit >= (int64_t)a.n_rows * per_row) return;
    const int r = (int)(unit / per_row), y = (int)(unit % per_row);
    const int kvh = y / chunks, g0 = y % chunks * G, h0 = kvh * a.group + g0;
    const int ng = min(G, a.group - g0);
    const int sub = lane / LPK, d0 = lane % LPK * DPL;
    const int pos = a.position[r];
    const int slot = a.k ? a.slot[r] : -1;
    int plen;
    const int pre = prefix_of(a, r, plen);
    // q, scaled, and the new row as the cache will hold it
    float q[G][DPL];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const float* const qr = a.q + r * a.ld_q + (h0 + min(g, ng - 1)) * kDim + d0;
#pragma unroll
        for (int d = 0; d < DPL; d += 4) {
            const f4 x = *reinterpret_cast<const f4*>(qr + d);
#pragma unroll
            for (int e = 0; e < 4; ++e) q[g][d + e] = __fmul_rn(x[e], a.scale);
        }
    }
    typename C::Raw new_k{}, new_v{};
    if (a.k) {
        const int64_t at = r * a.ld_kv + kvh * kDim + d0;
#pragma unroll
        for (int d = 0; d < DPL; d += 4) {
            const f4 x = *reinterpret_cast<const f4*>(a.k + at + d), z = *reinterpret_cast<const f4*>(a.v + at + d);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                new_k[d + e] = (T)x[e];
                new_v[d + e] = (T)z[e];
            }
        }
    }
    // keys [c0, c1) of the row: its own alone where tiles take the prefix
    const int cap = a.max_pages << a.shift;
    const int lo = a.tiles ? min(plen, pos + 1) : 0;
    const int end = min(pos + 1, plen + cap);
    const int L = max(end - lo, 0), used = min(a.n_own > 0 ? a.n_own : 1, (L + a.min_part - 1) / a.min_part);
    const int size = used > 0 ? (L + used - 1) / used : 0;
    const int c0 = lo + part * size, c1 = part < used ? min(c0 + size, end) : c0;
    const T* const kc = static_cast<const T*>(a.kc);
    const T* const vc = static_cast<const T*>(a.vc);
    // whether the new position is this part's, and one that the row sees
    const bool has_new = a.k && pos >= c0 && pos < c1;
    const uint32_t home = cache_row(a, slot < 0 ? -1 : slot >> a.shift, kvh, slot);
    if (has_new && home != kNoRow && g0 == 0 && sub == 0 && (W == 1 || w == 0)) {
        const uint64_t at = ((uint64_t)home << 6) + d0;
        *reinterpret_cast<typename C::Raw*>(const_cast<T*>(kc) + at) = new_k;
        *reinterpret_cast<typename C::Raw*>(const_cast<T*>(vc) + at) = new_v;
    }
    float o[G][DPL], m[G], s[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
#pragma unroll
        for (int d = 0; d < DPL; ++d) o[g][d] = 0.0f;
        m[g] = -INFINITY;
        s[g] = 0.0f;
    }
    const int32_t* const own_t = a.tables + (int64_t)r * a.max_pages;
    const int32_t* const pre_t = a.tables + (int64_t)max(pre, 0) * a.max_pages;
    for (int s0 = c0; s0 < c1;) {
        // the ids of [s0, s1): the prefix's pages, then the row's own, 64 in all
        const int a0 = s0 >> a.shift, b0 = (max(s0, plen) - plen) >> a.shift;
        const int n_pre = s0 < plen ? min(((min(c1, plen) - 1) >> a.shift) - a0 + 1, 64) : 0;
        const int64_t reach = n_pre > 0 && (int64_t)(a0 + n_pre) << a.shift < plen
                                  ? (int64_t)(a0 + n_pre) << a.shift
                                  : plen + ((int64_t)(b0 + 64 - n_pre) << a.shift);
        const int s1 = (int)min((int64_t)c1, reach);
        const int n_ids = n_pre + (s1 > plen ? ((s1 - 1 - plen) >> a.shift) - b0 + 1 : 0);
        const int32_t* const from = lane < n_pre ? pre_t + a0 + lane : own_t + b0 + lane - n_pre;
        const int held = lane < n_ids ? *from : -1;
        // a wave's batches of KPI kU keys in turn with the workgroup's
        for (int j0 = s0 + (W == 4 ? w * KPI * kU : 0); j0 < s1; j0 += W * KPI * kU) {
            typename C::Raw kk[kU], vv[kU];
            bool on[kU];
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const int j = min(j0 + KPI * u + sub, s1 - 1);
                const bool theirs = j < plen;
                const int place = theirs ? j : j - plen;
                const int id = __shfl(held, (place >> a.shift) - (theirs ? a0 : b0 - n_pre));
                const uint32_t row = cache_row(a, id, kvh, place);
                on[u] = j0 + KPI * u + sub < s1 && row != kNoRow;
                const uint64_t at = ((uint64_t)(row == kNoRow ? 0 : row) << 6) + d0;
                kk[u] = *reinterpret_cast<const typename C::Raw*>(kc + at);
                vv[u] = *reinterpret_cast<const typename C::Raw*>(vc + at);
            }
            if (has_new && pos >= j0 && pos < j0 + KPI * kU) {
#pragma unroll
                for (int u = 0; u < kU; ++u)
                    if (j0 + KPI * u + sub == pos) {
                        kk[u] = new_k;
                        vv[u] = new_v;
                        on[u] = home != kNoRow;
                    }
            }
            // a value that the row does not see may be anything: 0 instead
            bool all = true;
#pragma unroll
            for (int u = 0; u < kU; ++u) all = all && on[u];
            const bool whole = __ballot(!all) == 0;
            if (!whole) {
#pragma unroll
                for (int u = 0; u < kU; ++u)
                    if (!on[u]) vv[u] = typename C::Raw{};
            }
#pragma unroll
            for (int g = 0; g < G; ++g) {
                float x[kU], bm = -INFINITY;
#pragma unroll
                for (int u = 0; u < kU; ++u) {
                    float t = 0.0f;
#pragma unroll
                    for (int d = 0; d < DPL; ++d) t = __fmaf_rn(C::at(kk[u], d), q[g][d], t);
                    t = __fadd_rn(t, dpp16<0xB1>(t));  // the key's lanes
                    t = __fadd_rn(t, dpp16<0x4E>(t));
                    t = __fadd_rn(t, dpp16<0x141>(t));
                    if (LPK == 16) t = __fadd_rn(t, dpp16<0x140>(t));
                    x[u] = t;
                }
                if (!whole) {
#pragma unroll
                    for (int u = 0; u < kU; ++u) x[u] = on[u] ? x[u] : -INFINITY;
                }
#pragma unroll
                for (int u = 0; u < kU; ++u) bm = fmaxf(bm, x[u]);
                const float nr = fmaxf(m[g], __builtin_ceilf(bm));
                if (__ballot(nr > m[g])) {
                    const float f = rescale(m[g], nr);
                    s[g] = __fmul_rn(s[g], f);
#pragma unroll
                    for (int d = 0; d < DPL; ++d) o[g][d] = __fmul_rn(o[g][d], f);
                    m[g] = nr;
                }
                // a key that is not there, or -inf while none is larger, has weight 0
                const float off = m[g] == -INFINITY ? 0.0f : m[g];
#pragma unroll
                for (int u = 0; u < kU; ++u) {
                    const float e = __builtin_amdgcn_exp2f(__fsub_rn(x[u], off));
                    s[g] = __fadd_rn(s[g], e);
#pragma unroll
                    for (int d = 0; d < DPL; ++d) o[g][d] = __fmaf_rn(C::at(vv[u], d), e, o[g][d]);
                }
            }
        }
        s0 = s1;
    }
    // the lane groups joined: every group ends with the wave's (m, s, o)
#pragma unroll
    for (int g = 0; g < G; ++g) {
#pragma unroll
        for (int x = LPK; x < 64; x <<= 1) {
            const float mo = __shfl_xor(m[g], x), so = __shfl_xor(s[g], x);
            const float M = fmaxf(m[g], mo);
            const float f = rescale(m[g], M), fo = rescale(mo, M);
            s[g] = __fadd_rn(__fmul_rn(s[g], f), __fmul_rn(so, fo));
#pragma unroll
            for (int d = 0; d < DPL; ++d)
                o[g][d] = __fadd_rn(__fmul_rn(o[g][d], f), __fmul_rn(__shfl_xor(o[g][d], x), fo));
            m[g] = M;
        }
    }
    // head h0 + g of the row from 64 lanes, a dimension each: a part, or the row's
    const auto store = [&](int g, float pm, float ps, float po) {
        if (a.n_own > 0) {
            const int64_t at = ((int64_t)part * a.n_rows + r) * a.n_head + h0 + g;
            if (lane == 0) a.part_ms[at] = float2{pm, ps};
            if (c0 < c1) a.part_o[at * kDim + lane] = po;
        } else {
            attn_store(a.o, r, h0 + g, lane, ps == 0.0f ? 0.0f : __fdiv_rn(po, ps));
        }
    };
    __shared__ __align__(16) float red_o[4][G][kDim];
    if (sub == 0) {
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int d = 0; d < DPL; ++d) red_o[w][g][d0 + d] = o[g][d];
    }
    if constexpr (W == 1) {  // wave-private: its own stores are seen in order
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int g = 0; g < G; ++g)
            if (g < ng) store(g, m[g], s[g], red_o[w][g][lane]);
    } else {
        __shared__ float red_m[4][G], red_s[4][G];
        if (lane == 0) {
#pragma unroll
            for (int g = 0; g < G; ++g) {
                red_m[w][g] = m[g];
                red_s[w][g] = s[g];
            }
        }
        __syncthreads();
        for (int g = w; g < ng; g += 4) {
            float M = red_m[0][g];
#pragma unroll
            for (int i = 1; i < 4; ++i) M = fmaxf(M, red_m[i][g]);
            float st = 0.0f, ot = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float f = rescale(red_m[i][g], M);
                st = __fadd_rn(st, __fmul_rn(red_s[i][g], f));
                ot = __fadd_rn(ot, __fmul_rn(red_o[i][g][lane], f));
            }
            store(g, M, st, ot);
        }
    }
}

// ------------------------------------------------------------------ joins

// One wave per row and head: the row's own parts and its prefix's, 64 at a
// time: a lane each for maxima and sums, then each quarter of the wave every
// fourth part's values, four to a lane and four loads in flight (one part after
// the other, 64 lanes a part: 6.6 us behind one row's parts where this takes 3.7).
__global__ __launch_bounds__(256) void kv_join(KvArgs a) {
    const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const int64_t x = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (x >= (int64_t)a.n_rows * a.n_head) return;
    const int r = (int)(x / a.n_head), h = (int)(x % a.n_head);
    const int64_t rows = (int64_t)a.n_rows * a.n_head;
    const int most = a.n_own + a.n_shared;
    float2 ms = a.part_ms[min(lane, most - 1) * rows + x];
    int plen;
    prefix_of(a, r, plen);
    // parts of this row: none without a position
    const bool live = a.position[r] >= 0;
    const int n = live ? a.n_own + (plen > 0 ? a.n_shared : 0) : 0;
    float M = -INFINITY, st = 0.0f;
    f4 ot = f4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int p0 = 0; p0 < n; p0 += 64) {
        if (p0 > 0) ms = a.part_ms[min(p0 + lane, most - 1) * rows + x];
        if (p0 + lane >= n) ms = float2{-INFINITY, 0.0f};
        float bm = ms.x;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) bm = fmaxf(bm, __shfl_xor(bm, o));
        const float nm = fmaxf(M, bm);
        const float keep = rescale(M, nm);
        st = __fmul_rn(st, keep);
        ot *= keep;
        M = nm;
        // a part that saw nothing has no values: they are not read into the sum
        const uint64_t some = __ballot(!(ms.y == 0.0f));
        const float f = rescale(ms.x, M);
        float sf = some >> lane & 1 ? __fmul_rn(ms.y, f) : 0.0f;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) sf = __fadd_rn(sf, __shfl_xor(sf, o));
        st = __fadd_rn(st, sf);
        const int last = some ? 64 - (int)__builtin_clzll(some) : 0;
        for (int i0 = 0; i0 < last; i0 += 16) {
            f4 y[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
                y[u] = *reinterpret_cast<const f4*>(
                    a.part_o + ((p0 + min(i0 + 4 * u + g, last - 1)) * rows + x) * kDim + 4 * c);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int i = i0 + 4 * u + g;
                const float fi = __shfl(f, i);
                if (some >> i & 1) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) ot[e] = __fadd_rn(ot[e], __fmul_rn(y[u][e], fi));
                }
            }
        }
    }
#pragma unroll
    for (int o = 16; o < 64; o <<= 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) ot[e] = __fadd_rn(ot[e], __shfl_xor(ot[e], o));
    const float over = st == 0.0f ? 0.0f : __fdiv_rn(1.0f, st);
    attn_store4(a.o, a.n_rows, g == 0 ? r : a.n_rows, h, c, ot * over);
}

// ------------------------------------------------------------------ tiles

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
// addresses chosen among several are kept as ones of device memory
typedef const __attribute__((address_space(1))) u4* global_u4;
typedef const __attribute__((address_space(1))) int32_t* global_i32;
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

// Values as parts that the 16-bit matrix cores multiply exactly (products in
// fp32), two to a dword.
//  * fp32 caches: three bf16 parts, each the leading 8 bits of what the ones
//    before leave: x = h + m + l to the last bit wherever l is not subnormal,
//    at any magnitude.  Of the nine products of two such values six are formed:
//    |m| < 2^-7 |x| and |l| < 2^-15 |x|, so m l + l m + l l is below 2^-21 of the
//    whole (and 2^-24 of it on average).
//  * fp16 caches: keys and values as they are; queries and weights two fp16
//    parts, x = hi + lo to 2^-22.
// The fp32 matrix instructions run on the vector units' own multipliers, 32
// cycles for a 16x16x4, and nothing else runs beside them: with them the
// softmax's vector work came on top (us, prefix part of 512 rows x 2001 keys x
// 16 heads: 67; prompts of 64 x 129-383 rows: 236).
template <class T>
struct Parts;
template <>
struct Parts<float> {
    static constexpr int kKv = 3, kQ = 3, kProducts = 6;
    __device__ static constexpr int kv(int i) { constexpr int x[6] = {2, 1, 0, 1, 0, 0}; return x[i]; }
    __device__ static constexpr int q(int i) { constexpr int x[6] = {0, 1, 2, 0, 1, 0}; return x[i]; }
    // parts of two neighbours
    __device__ static __forceinline__ void split(float x, float y, uint32_t (&p)[3]) {
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            const uint32_t u = __builtin_bit_cast(uint32_t, x), v = __builtin_bit_cast(uint32_t, y);
            p[i] = __builtin_amdgcn_perm(v, u, 0x07060302u);  // their upper halves
            x = __fsub_rn(x, __builtin_bit_cast(float, u & 0xffff0000u));
            y = __fsub_rn(y, __builtin_bit_cast(float, v & 0xffff0000u));
        }
    }
    __device__ static __forceinline__ void split_weights(float x, float y, uint32_t (&p)[3]) { split(x, y, p); }
    static constexpr uint32_t kOnes = 0x3f803f80;
    __device__ static __forceinline__ f4 mfma(const u4& x, const u4& y, const f4& acc) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, x),
                                                       __builtin_bit_cast(b8, y), acc, 0, 0, 0);
    }
};
template <>
struct Parts<_Float16> {
    static constexpr int kKv = 1, kQ = 2, kProducts = 2;
    __device__ static constexpr int kv(int) { return 0; }
    __device__ static constexpr int q(int i) { return 1 - i; }
    __device__ static __forceinline__ void split(float x, float y, uint32_t (&p)[2]) {
        const _Float16 a = (_Float16)x, b = (_Float16)y;
        p[0] = __builtin_bit_cast(uint32_t, split_h2{a, b});
        p[1] = __builtin_bit_cast(uint32_t, split_h2{(_Float16)__fsub_rn(x, (float)a),
                                                     (_Float16)__fsub_rn(y, (float)b)});
    }
    // the weights': to 2^-20, both parts cut off instead of rounded (half the
    // operations); what is cut leaves their sum too, which is taken of the parts
    __device__ static __forceinline__ void split_weights(float x, float y, uint32_t (&p)[2]) {
        p[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x, y));
        const split_h2 h = __builtin_bit_cast(split_h2, p[0]);
        float one;  // opaque, for the mixed-precision form of x - hi
        asm("v_mov_b32 %0, 1.0" : "=v"(one));
        p[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(
                                                __fmaf_rn(-(float)h[0], one, x), __fmaf_rn(-(float)h[1], one, y)));
    }
    static constexpr uint32_t kOnes = 0x3c003c00;
    __device__ static __forceinline__ f4 mfma(const u4& x, const u4& y, const f4& acc) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, x),
                                                      __builtin_bit_cast(h8, y), acc, 0, 0, 0);
    }
};

// The largest of v over the four lanes of a 16-lane column (lane, lane ^ 16,
// lane ^ 32, lane ^ 48).
__device__ __forceinline__ float max_column(float v) {
    const uint32_t x = __builtin_bit_cast(uint32_t, v);
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    // the median with infinity: a maximum without a maximum's quieting of its operands
    const float m = __builtin_amdgcn_fmed3f(__builtin_bit_cast(float, (uint32_t)a[0]),
                                            __builtin_bit_cast(float, (uint32_t)a[1]), INFINITY);
    const uint32_t y = __builtin_bit_cast(uint32_t, m);
    const auto b = __builtin_amdgcn_permlane32_swap(y, y, false, false);
    return __builtin_amdgcn_fmed3f(__builtin_bit_cast(float, (uint32_t)b[0]),
                                   __builtin_bit_cast(float, (uint32_t)b[1]), INFINITY);
}

// Four keys of one dimension from rows of 16-bit values in LDS: of each 16
// lanes, lane 4 r + q names 4 dimensions (quarter q of 16) of key r, and lane i
// gets dimension i of keys 0 .. 3.
__device__ __forceinline__ u2 read_transposed(const char* p) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s4 lds_s4;
    return __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p)));
}

// A tile's walk: [0, plen) in pre_t's pages, the rest in own_t's, from
// position fresh0 on the call's own rows from row fresh_row (which its streams
// store in this launch).
struct Walk {
    const int32_t* pre_t;
    const int32_t* own_t;
    int plen, end, fresh0, fresh_row;
};

// 16 (row, head) pairs of a tile a wave, on the matrix cores.  The keys and
// values of a stage (kKeys of them) are loaded once for the workgroup, through
// registers into LDS (as parts) while the stage before is computed on; their
// places are looked up a stage before that.
//  * Scores transposed, S^T = K Q^T, 32 keys at a time: lane (g = l / 16,
//    c = l % 16) ends with pair c's scores at keys 4 g + i and 16 + 4 g + i, so
//    a pair's limit, maximum, sum and rescaling are its own lanes', joined over
//    g by two exchanges.
//  * Outputs transposed, O^T = V^T P^T: those weights are the second operand as
//    they stand, V's operand is read transposed (tile dt: dimension 16 dt +
//    4 g + i).
// With fp16 parts q is scaled by a power of two per pair (its largest magnitude
// to [2^14, 2^15)) and the weights by 2^14 (their largest is 1), so that parts
// lose nothing to subnormals that the sum would notice.
// A key that a pair does not see has weight 0, and 0 times a V that is not
// finite would reach the pair: a stage that holds such values is noted as it is
// stored, and where some pair does not see all of 32 keys of it, they are added
// pair by pair with the unseen keys' V at 0.
// SPLIT: the four waves take the same 16 pairs and 32 keys of a stage each,
// joined through LDS (few rows); else each wave its own pairs and all keys.
// FORM: the prompt form; the step form's prefixes, keys cut over workgroups,
// parts stored; or one row's heads of a key head against the row's keys, cut
// likewise (where many query heads share a key head: the step form on the
// vector units then spends its time on products).
// Prompts of 4 x 4096 rows take fp32 965 to 990 us (139 to 142 TFLOP/s of the
// formula's, six times as many of the parts' without the weights' sums), fp16 525
// (262, twice as many): the vector units' instructions (half the time fp32, 60 %
// fp16) and the matrix cores' (43 %, 30 %) together.  64 prompts of 129 to 383 rows
// fp32 130 us, 3.1 TB/s; 8 of 301 to 1501 fp16 behind 377 keys 125.  What made them faster: loads that stand behind the choice of their
// addresses (fp16 8 %), the longest tiles first (7 %), four workgroups a CU for
// fp16 (8 %), nothing kept over the loop that its end can find again (up to
// 7 %).  What did not: fewer instructions for a stage's addresses, all of K's
// reads before the products, 8 waves a workgroup, two sets of pairs a wave, 32
// pairs a wave on 32x32 products (804 us where these take 530).
enum { kPrompt, kPrefix, kOneRow };

// Tile t of prompts that come without a list of them, as the plan would have
// written it (count 0 or less: none): stream i's tiles have the numbers from
// row_start[i] / tile_rows + i on, so none of them reaches the next stream's first
// and t is below n_rows / tile_rows + n_streams.  Every lane of the wave takes
// part: 64 streams are tried at a time.
__device__ __forceinline__ int4 tile_of(const KvArgs& a, int t) {
    const int lane = threadIdx.x & 63, T = a.tile_rows;
    int i = 0, end = a.n_streams;
    while (end - i > 1) {  // the last stream of [i, end) whose first number is at most t
        const int step = (end - i + 63) / 64, x = i + lane * step;
        const bool on = x < end && a.row_start[min(x, end - 1)] / T + x <= t;
        i += max((int)__popcll(__ballot(on)) - 1, 0) * step;
        end = min(i + step, end);
    }
    const int r0 = a.row_start[i], r1 = min(a.row_start[i + 1], a.n_rows);
    const int first = min(max(r0 + (t - r0 / T - i) * T, 0), a.n_rows), count = min(T, r1 - first);
    return make_int4(i, first, count, count > 0 ? a.position[first + count - 1] + 1 : 0);
}

template <class T, bool SPLIT, int FORM>
__device__ __forceinline__ void tiles_of(const KvArgs& a, uint32_t block, uint32_t blocks, int cut) {
    constexpr bool F16 = sizeof(T) == 2, PROMPT = FORM == kPrompt;
    static_assert(SPLIT || FORM != kOneRow, "a row's heads are one wave's pairs");
    constexpr int kKeys = SPLIT ? 128 : 32;
    using P = Parts<T>;
    constexpr int kCh = kDim * sizeof(T) / 16;       // 16-byte chunks of a row in memory
    constexpr int kStep = 256 / kCh;                 // rows that the workgroup loads at a time
    constexpr int kU = kKeys / kStep;               // rows a thread loads of a stage
    static_assert(kStep % 16 == 0, "a thread's rows have one order of chunks");
    constexpr int kPer = 16 / sizeof(T);             // values of a chunk
    constexpr int kPad = kDim + 4;                   // a pair's outputs in LDS
    constexpr int kPart = kKeys * kDim * 2, kStage = P::kKv * kPart;  // bytes: a part, K or V
    constexpr int kBufs = SPLIT ? 1 : 2;
    // [buffer][K, V][part], then the outputs in their place
    constexpr int kOut = 4 * 16 * kPad * 4, kLds = 2 * kBufs * kStage;
    __shared__ __align__(16) char lds[kLds > kOut ? kLds : kOut];
    // of a stage (three in turn: one read, one written, one cleared): whether
    // values are not finite, and the keys without a place, a bit each
    __shared__ int odd[3];
    __shared__ uint32_t gone[3][kKeys / 32];
    __shared__ float join_m[4][16], join_s[4][16];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int g = lane >> 4, c = lane & 15;
    const int kvh = block % a.n_kv, unit = block / a.n_kv;
    const T* const kc = static_cast<const T*>(a.kc);
    const T* const vc = static_cast<const T*>(a.vc);
    const auto dead_rows = [&]() {  // rows behind the last give zeros
        if (!PROMPT) return;
        const int total = a.row_start[a.n_streams];
        for (int64_t r = (int64_t)max(total, 0) + block; r < a.n_rows; r += blocks)
            for (int h = w; h < a.n_head; h += 4) attn_store(a.o, (int)r, h, lane, 0.0f);
    };
    // the workgroup's rows: [first, first + count) of the call (of order, where
    // prefixes are shared) for key stream `who`, and its first pair
    const int subs = FORM == kOneRow ? (a.group + 15) / 16 : 4;
    const int p0 = SPLIT ? 16 * (unit % subs) : 0;
    int who, first, count, keys;
    if (FORM == kOneRow) {
        who = first = unit / subs;
        count = 1;
        keys = 0;
    } else {
        const int t = PROMPT ? a.n_tiles - 1 - (SPLIT ? unit / 4 : unit) : unit;
        const int4 tile = PROMPT && !a.tiles ? tile_of(a, t) : a.tiles[t];
        who = __builtin_amdgcn_readfirstlane(tile.x);
        first = min(max(__builtin_amdgcn_readfirstlane(tile.y), 0), a.n_rows);
        count = min(__builtin_amdgcn_readfirstlane(tile.z), a.tile_rows);
        keys = __builtin_amdgcn_readfirstlane(tile.w);
        if (who < 0 || who >= a.n_streams) count = 0;
    }
    const int pairs = count * a.group;
    if (p0 >= pairs) {
        dead_rows();
        return;
    }
    // the row of a lane's pair (-1: none), its query head
    const auto pair_of = [&](int lane_of, int& h, int wave) {
        const int p = p0 + (SPLIT ? 0 : 16 * wave) + (lane_of & 15);
        const int local = over_group(a, p), at = first + local;
        h = kvh * a.group + p - local * a.group;
        int row = -1;
        if (p < pairs && at < a.n_rows) row = FORM == kPrefix ? a.order[at] : at;
        return row < a.n_rows ? row : -1;
    };
    int h;
    const int row = pair_of(lane, h, w);
    const bool real = row >= 0;
    const int rc = real ? row : 0;
    // the walk, and lim, the last key the pair sees
    const int cap = a.max_pages << a.shift;
    Walk k;
    int lim, begin = 0;
    k.own_t = a.tables + (int64_t)who * a.max_pages;
    k.pre_t = k.own_t;
    k.fresh0 = INT32_MAX;
    k.fresh_row = 0;
    if (FORM == kPrefix) {
        k.plen = 0;
        prefix_of(a, rc, lim);
        lim = real ? lim - 1 : -1;
        // this workgroup's keys, the same for all pairs of the tile
        keys = min(max(keys, 0), cap);
        const int used = min(a.n_shared, (keys + 63) / 64);
        const int size = used > 0 ? ((keys + used - 1) / used + 31) / 32 * 32 : 0;
        begin = min(cut * size, keys);
        k.end = min(begin + size, keys);
    } else {
        const int pre = prefix_of(a, who, k.plen);
        if (pre >= 0) k.pre_t = a.tables + (int64_t)pre * a.max_pages;
        lim = real ? min(a.position[rc], k.plen + cap - 1) : -1;
        k.end = min(keys, k.plen + cap);
        if (PROMPT && a.k) {  // the stream's first new row and its position
            k.fresh_row = min(max(a.row_start[who], 0), first);
            k.fresh0 = max(a.position[min(first, a.n_rows - 1)] - (first - k.fresh_row), 0);
        }
        // with SPLIT, the pairs' last key ends the walk
        if (PROMPT && SPLIT) {
            const int end_row = first + over_group(a, min(p0 + 15, pairs - 1));
            k.end = min(k.end, a.position[min(end_row, a.n_rows - 1)] + 1);
        }
        if (FORM == kOneRow) {  // a part of the row's keys: its own alone where tiles take the prefix
            const int pos = a.position[first], stop = min(pos + 1, k.plen + cap);
            begin = a.tiles ? min(k.plen, pos + 1) : 0;
            const int L = max(stop - begin, 0);
            const int used = min(max(a.n_own, 1), (L + a.min_part - 1) / a.min_part);
            const int size = used > 0 ? ((L + used - 1) / used + 31) / 32 * 32 : 0;
            begin = min(begin + cut * size, max(stop, 0));
            k.end = min(begin + size, stop);
            // the new row to its slot before it is read with the others
            if (a.k && pos >= begin && pos < k.end) {
                const int slot = a.slot[first];
                const uint32_t home = cache_row(a, slot < 0 ? -1 : slot >> a.shift, kvh, slot);
                if (home != kNoRow && tid < 16) {
                    const int64_t x = first * a.ld_kv + kvh * kDim + 4 * tid;
                    store4(const_cast<T*>(kc), home, 4 * tid, *reinterpret_cast<const f4*>(a.k + x));
                    store4(const_cast<T*>(vc), home, 4 * tid, *reinterpret_cast<const f4*>(a.v + x));
                }
                __syncthreads();
            }
        }
    }
    k.end = __builtin_amdgcn_readfirstlane(k.end);  // as the whole workgroup has it
    k.plen = __builtin_amdgcn_readfirstlane(k.plen);
    k.fresh0 = __builtin_amdgcn_readfirstlane(k.fresh0);
    k.fresh_row = __builtin_amdgcn_readfirstlane(k.fresh_row);
    begin = __builtin_amdgcn_readfirstlane(begin);
    // a part in LDS: rows of eight 16-byte chunks, a row's in an order of its own
    // so that 16 rows' reads of one chunk fall in different banks
    const auto chunk_at = [](int r, int ch) { return (r * 8 + (ch ^ (r >> 1 & 7))) * 16; };
    const int ch = tid % kCh, r0 = tid / kCh;
    int next[kU];
    // a stage's loads, nothing of them used before they are stored: a chunk of
    // K and V each, the fp16 forms' new rows (fp32) in two
    constexpr int kLoads = F16 && PROMPT ? 2 : 1;
    u4 kr[kU][kLoads], vr[kU][kLoads];
    uint32_t none = 0, fresh = 0;  // rows that have no place, and new ones: a bit each
    bool some_new = false;  // in the stage, and so for the workgroup
    // the tile's own new rows (with SPLIT, those that begin among its pairs) go to
    // their slots as they are staged: rows [own0, own1) of the call
    uint32_t to[kU];
    const int own0 = !PROMPT || !a.k ? 0 : first + over_group(a, p0 + a.group - 1);
    const int own1 = !PROMPT || !a.k ? 0 : min(first + min(SPLIT ? over_group(a, p0 + 15 + a.group) : count, count), a.n_rows);
    // the table entry that says where key j < end is (a new row's: its slot).  Here
    // and in load the addresses may come by a branch, the loads themselves stand
    // after it: a load on one side alone is waited for where the sides meet.
    const auto look = [&](int j0) {
        const int32_t* from[kU];
        if (PROMPT && j0 >= k.fresh0) {  // the call's own rows alone
            const int r = k.fresh_row + (j0 - k.fresh0) + r0;
#pragma unroll
            for (int u = 0; u < kU; ++u) from[u] = a.slot + min(r + u * kStep, a.n_rows - 1);
        } else {
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const int x = min(j0 + r0 + u * kStep, k.end - 1);
                const bool theirs = x < k.plen;
                from[u] = (theirs ? k.pre_t : k.own_t) + ((theirs ? x : x - k.plen) >> a.shift);
                if (PROMPT && x >= k.fresh0) from[u] = a.slot + min(k.fresh_row + (x - k.fresh0), a.n_rows - 1);
            }
        }
#pragma unroll
        for (int u = 0; u < kU; ++u) next[u] = *(global_i32)from[u];
    };
    // the stage from j0 on, its entries in next
    const uint32_t places = (uint32_t)a.n_pages << a.shift, in_page = (1u << a.shift) - 1;
    const auto load = [&](int j0) {
        none = fresh = 0;
        const char *ks[kU], *vs[kU];
        const int rf = k.fresh_row + (j0 - k.fresh0);  // the stage's first row, where all are new
        some_new = PROMPT && j0 + kKeys > k.fresh0;
        if (PROMPT && j0 >= k.fresh0) {
            fresh = (1u << kU) - 1;
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const int r = min(rf + r0 + u * kStep, a.n_rows - 1);
                none |= (uint32_t)(j0 + r0 + u * kStep >= k.end || (uint32_t)next[u] >= places) << u;
                const uint64_t from = (uint64_t)(uint32_t)r * (uint32_t)a.ld_kv + (kvh * kDim + kPer * ch);
                ks[u] = reinterpret_cast<const char*>(a.k + from);
                vs[u] = reinterpret_cast<const char*>(a.v + from);
                to[u] = kNoRow;
            }
            if (rf < own1 && rf + kKeys > own0) {
#pragma unroll
                for (int u = 0; u < kU; ++u) {
                    const int r = rf + r0 + u * kStep;
                    const uint32_t row = (((uint32_t)(next[u] >> a.shift) * (uint32_t)a.n_kv + (uint32_t)kvh)
                                          << a.shift) + ((uint32_t)next[u] & in_page);
                    to[u] = !(none >> u & 1) && r >= own0 && r < own1 ? row : kNoRow;
                }
            }
        } else {
            const auto places_of = [&](auto mixed) {
#pragma unroll
                for (int u = 0; u < kU; ++u) {
                    const int j = j0 + r0 + u * kStep;
                    const bool own = mixed && j >= k.fresh0;
                    const int page = own ? next[u] >> a.shift : next[u];
                    const int off = own ? next[u] : j < k.plen ? j : j - k.plen;
                    const bool there = (uint32_t)page < (uint32_t)a.n_pages;
                    uint32_t row = (((uint32_t)page * (uint32_t)a.n_kv + (uint32_t)kvh) << a.shift) +
                                   ((uint32_t)off & in_page);
                    row = there ? row : 0;
                    none |= (uint32_t)(j >= k.end || !there) << u;
                    const uint64_t from = (uint64_t)row << 6;
                    ks[u] = reinterpret_cast<const char*>(kc + kPer * ch + from);
                    vs[u] = reinterpret_cast<const char*>(vc + kPer * ch + from);
                    to[u] = kNoRow;
                    if (mixed) {
                        fresh |= (uint32_t)own << u;
                        const int r = min(k.fresh_row + (j - k.fresh0), a.n_rows - 1);
                        const uint64_t x = (uint64_t)(uint32_t)r * (uint32_t)a.ld_kv + (kvh * kDim + kPer * ch);
                        ks[u] = own ? reinterpret_cast<const char*>(a.k + x) : ks[u];
                        vs[u] = own ? reinterpret_cast<const char*>(a.v + x) : vs[u];
                        to[u] = own && !(none >> u & 1) && r >= own0 && r < own1 ? row : kNoRow;
                    }
                }
            };
            if (some_new) places_of(std::true_type());
            else places_of(std::false_type());
        }
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            kr[u][0] = *(global_u4)(ks[u]);
            vr[u][0] = *(global_u4)(vs[u]);
            if (kLoads == 2) {  // a new row's other half; a cached chunk again
                const int more = fresh >> u & 1 ? 16 : 0;
                kr[u][kLoads - 1] = *(global_u4)(ks[u] + more);
                vr[u][kLoads - 1] = *(global_u4)(vs[u] + more);
            }
        }
    };
    const auto store = [&](int b, int slot) {
        char* const kb = lds + 2 * b * kStage;
        if (__ballot(none != 0)) {
#pragma unroll
            for (int u = 0; u < kU; ++u)
                if (none >> u & 1) {
                    if (ch == 0) atomicOr(&gone[slot][(r0 + u * kStep) >> 5], 1u << ((r0 + u * kStep) & 31));
                    kr[u][0] = vr[u][0] = u4{0, 0, 0, 0};
                    if (F16 && PROMPT) kr[u][kLoads - 1] = vr[u][kLoads - 1] = u4{0, 0, 0, 0};
                }
        }
        // 0 times every value: NaN once one is not finite
        float odd4 = 0.0f;
        split_h2 odd8 = split_h2{(_Float16)0.0f, (_Float16)0.0f};
#pragma unroll
        for (int u = 0; u < kU; ++u) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {  // K, V
                u4 y = x ? vr[u][0] : kr[u][0];
                if constexpr (F16 && PROMPT) {
                    if (some_new && (fresh >> u & 1)) {  // rounded as the cache will hold them
                        const f4 lo = __builtin_bit_cast(f4, y);
                        const f4 hi = __builtin_bit_cast(f4, x ? vr[u][1] : kr[u][1]);
                        y = __builtin_bit_cast(u4, h8{(_Float16)lo[0], (_Float16)lo[1], (_Float16)lo[2],
                                                      (_Float16)lo[3], (_Float16)hi[0], (_Float16)hi[1],
                                                      (_Float16)hi[2], (_Float16)hi[3]});
                    }
                }
                if (PROMPT && some_new && to[u] != kNoRow)
                    *reinterpret_cast<u4*>(const_cast<T*>(x ? vc : kc) + ((uint64_t)to[u] << 6) + kPer * ch) = y;
                if constexpr (F16) {
                    if (x) {
                        const split_h2 zero = split_h2{(_Float16)0.0f, (_Float16)0.0f};
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            odd8 = __builtin_elementwise_fma(__builtin_bit_cast(split_h2, (uint32_t)y[i]), zero, odd8);
                    }
                    *reinterpret_cast<u4*>(kb + (chunk_at(r0, ch) + u * (kStep * 128) + x * kStage)) = y;
                } else {
                    const f4 z = __builtin_bit_cast(f4, y);
                    if (x) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) odd4 = __fmaf_rn(z[i], 0.0f, odd4);
                    }
                    uint32_t lo[P::kQ], hi[P::kQ];
                    P::split(z[0], z[1], lo);
                    P::split(z[2], z[3], hi);
#pragma unroll
                    for (int i = 0; i < P::kKv; ++i)
                        *reinterpret_cast<u2*>(kb + (chunk_at(r0, ch >> 1) + 8 * (ch & 1) +
                                                     u * (kStep * 128) + x * kStage + i * kPart)) = u2{lo[i], hi[i]};
                }
            }
        }
        if (F16) odd4 = (float)odd8[0] + (float)odd8[1];
        if (odd4 != odd4) odd[slot] = 1;
    };
    // q, scaled: dimensions 32 ks + 8 g .. of pair c, in parts; c2: the power of two
    // that a score as the matrix cores give it is short of
    u4 qp[2][P::kQ];
    float c2 = 1.0f;
    {
        const float* const qr = a.q + rc * a.ld_q + (real ? h : 0) * kDim;
        float x[2][8], mx = 0.0f;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const f4 v = *reinterpret_cast<const f4*>(qr + 32 * ks + 8 * g + e) * a.scale;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[ks][e + i] = v[i];
                    mx = fmaxf(mx, fabsf(v[i]));
                }
            }
        float sc = 1.0f;
        if (F16) {
            mx = max_column(mx);
            split_scale(mx, sc, c2);
        }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint32_t y[P::kQ];
                P::split(__fmul_rn(x[ks][2 * e], sc), __fmul_rn(x[ks][2 * e + 1], sc), y);
#pragma unroll
                for (int i = 0; i < P::kQ; ++i) qp[ks][i][e] = y[i];
            }
    }
    // the weights' scale, a power of two, and how far one may pass it: with fp16
    // parts by 2 (below 65504)
    constexpr float kUp = F16 ? 14.0f : 0.0f, kSlack = F16 ? 1.0f : 16.0f;
    f4 o[4];
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) o[dt] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    // the reference, negated (kUp below the largest exponent when it was chosen), and
    // how far over it an exponent moves it (-inf: no key yet)
    float off = 0.0f, bar = -INFINITY;
    f4 sum = f4{0.0f, 0.0f, 0.0f, 0.0f};  // the first of it
    int last = lim, least = real ? lim : INT32_MAX;
    const auto over = [&](auto x) {  // lanes at a distance of x
        last = max(last, __builtin_amdgcn_ds_swizzle(last, x << 10 | 0x1f));
        least = min(least, __builtin_amdgcn_ds_swizzle(least, x << 10 | 0x1f));
    };
    over(std::integral_constant<int, 1>());
    over(std::integral_constant<int, 2>());
    over(std::integral_constant<int, 4>());
    over(std::integral_constant<int, 8>());
    last = __builtin_amdgcn_readfirstlane(last);
    least = __builtin_amdgcn_readfirstlane(least);

    // the lane's chunks of a buffer's first 16 rows: K's of key c, V's four
    // dimensions of key 4 g + c / 4 (read_transposed)
    int k_at[2], v_at[4];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) k_at[ks] = chunk_at(c, 4 * ks + g);
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) v_at[dt] = chunk_at(4 * g + (c >> 2), 2 * dt + (c >> 1 & 1)) + 8 * (c & 1);

    // 32 keys from j0 on: rows b .. of a buffer
    const auto compute = [&](int buf, int slot, int b, int j0) {
        const char* const kb = lds + 2 * buf * kStage + b * 128;  // 32 rows on, the order is the same
        const uint32_t miss = __builtin_amdgcn_readfirstlane(gone[slot][b >> 5]);
        f4 x[2] = {f4{0.0f, 0.0f, 0.0f, 0.0f}, f4{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            u4 y[2][P::kKv];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int i = 0; i < P::kKv; ++i)
                    y[kt][i] = *reinterpret_cast<const u4*>(kb + k_at[ks] + (i * kPart + kt * 2048));
#pragma unroll
            for (int i = 0; i < P::kProducts; ++i)
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
                    x[kt] = P::mfma(y[kt][P::kv(i)], qp[ks][P::q(i)], x[kt]);
        }
        // whether some pair of the wave does not see all 32
        const bool partial = j0 + 31 > least || j0 + 32 > k.end || miss != 0;
        // the keys up to `limit` that are there, a bit each
        const auto seen = [&](int limit) {
            const int n = min(limit, k.end - 1) - j0;
            return (n < 0 ? 0u : n >= 31 ? ~0u : (2u << n) - 1) & ~miss;
        };
        if (partial) {
            const uint32_t see = seen(lim) >> (4 * g);
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (!(see >> (16 * kt + i) & 1)) x[kt][i] = -INFINITY;
        }
        // exponents by the pair's reference (0 before it has one); a larger one than
        // kUp + kSlack over it moves the reference up
        float top = -INFINITY;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[kt][i] = __fmaf_rn(x[kt][i], c2, off);
                top = fmaxf(top, x[kt][i]);
            }
        top = max_column(top);
        const bool move = top > bar;
        if (__ballot(move)) {
            const float to = move ? __fsub_rn(off, __fsub_rn(__builtin_ceilf(top), kUp)) : off;
            const float by = __fsub_rn(off, to);  // as far as it moves, once rounded
            const float f = bar == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(-by);
            off = to;
            if (move) bar = kUp + kSlack;
            sum[0] = __fmul_rn(sum[0], f);
#pragma unroll
            for (int dt = 0; dt < 4; ++dt)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[dt][i] = __fmul_rn(o[dt][i], f);
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int i = 0; i < 4; ++i) x[kt][i] = __fsub_rn(x[kt][i], by);
        }
        // weights; unseen keys and scores of -inf have none
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[kt][i] = __builtin_amdgcn_exp2f(x[kt][i]);
        const bool plain = !(partial && __builtin_amdgcn_readfirstlane(odd[slot]));
        u4 wp[P::kQ];  // the weights' parts, the lane's eight keys
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            uint32_t y[P::kQ];
            P::split_weights(x[e >> 1][2 * (e & 1)], x[e >> 1][2 * (e & 1) + 1], y);
#pragma unroll
            for (int i = 0; i < P::kQ; ++i) wp[i][e] = y[i];
        }
        // their sum, of the parts: every row of the product with ones
#pragma unroll
        for (int i = P::kQ - 1; i >= 0; --i)
            sum = P::mfma(u4{P::kOnes, P::kOnes, P::kOnes, P::kOnes}, wp[i], sum);
        const auto value = [&](int dt, int i) {  // part i of dimension 16 dt + c of the lane's keys
            u4 y;
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                const u2 z = read_transposed(kb + v_at[dt] + (kStage + i * kPart + kt * 2048));
                y[2 * kt] = z[0];
                y[2 * kt + 1] = z[1];
            }
            return y;
        };
        if (plain) {
#pragma unroll
            for (int dt = 0; dt < 4; ++dt) {
                u4 y[P::kKv];
#pragma unroll
                for (int i = 0; i < P::kKv; ++i) y[i] = value(dt, i);
#pragma unroll
                for (int i = 0; i < P::kProducts; ++i) o[dt] = P::mfma(y[P::kv(i)], wp[P::q(i)], o[dt]);
            }
        } else {
#pragma unroll 1
            for (int n = 0; n < 16; ++n) {
                const uint32_t see = seen(__builtin_amdgcn_readlane(lim, n)) >> (4 * g);
#pragma unroll
                for (int dt = 0; dt < 4; ++dt) {
                    u4 y[P::kKv];
#pragma unroll
                    for (int i = 0; i < P::kKv; ++i) {
                        y[i] = value(dt, i);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t two = see >> (16 * (e >> 1) + 2 * (e & 1));
                            y[i][e] &= (two & 1 ? 0xffffu : 0u) | (two & 2 ? 0xffff0000u : 0u);
                        }
                    }
                    f4 add = o[dt];
#pragma unroll
                    for (int i = 0; i < P::kProducts; ++i) add = P::mfma(y[P::kv(i)], wp[P::q(i)], add);
                    if (c == n) o[dt] = add;
                }
            }
        }
    };

    const int stages = (max(k.end - begin, 0) + kKeys - 1) / kKeys;
    if (tid < 3) {
        odd[tid] = 0;
#pragma unroll
        for (int i = 0; i < kKeys / 32; ++i) gone[tid][i] = 0;
    }
    __syncthreads();
    if (stages > 0) {
        look(begin);
        load(begin);
        look(begin + kKeys);
        store(0, 0);
    }
    __syncthreads();
    for (int t = 0; t < stages; ++t) {
        const int j0 = begin + t * kKeys, slot = t % 3;
        const bool more = t + 1 < stages;
        if (more) {
            load(j0 + kKeys);
            look(j0 + 2 * kKeys);
        }
        if (tid == 0) {
            odd[(t + 2) % 3] = 0;
#pragma unroll
            for (int i = 0; i < kKeys / 32; ++i) gone[(t + 2) % 3][i] = 0;
        }
#pragma unroll 1
        for (int b = SPLIT ? 32 * w : 0; b < kKeys; b += SPLIT ? kKeys : 32)
            if (j0 + b <= last && j0 + b < k.end) compute(kBufs == 2 ? t & 1 : 0, slot, b, j0 + b);
        if (kBufs == 1) __syncthreads();
        if (more) store(kBufs == 2 ? (t + 1) & 1 : 0, (t + 1) % 3);
        __syncthreads();
    }
    // what the lane stands for once more: kept over the loop it would cost registers
    int tid_end = tid;
    asm volatile("" : "+v"(tid_end));
    const int ge = tid_end >> 4 & 3, ce = tid_end & 15, we = tid_end >> 6;
    int h_end;
    const int row_end = pair_of(tid_end & 63, h_end, we);
    // through LDS into rows: [16 w + pair][dimension]
    float* const os = reinterpret_cast<float*>(lds) + 16 * we * kPad;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        *reinterpret_cast<f4*>(os + ce * kPad + 16 * i + 4 * ge) = o[i];
    }
    if (ge == 0) {
        join_m[we][ce] = bar == -INFINITY ? -INFINITY : -off;
        join_s[we][ce] = sum[0];
    }
    __syncthreads();
    // lane (g, c): dimensions 4 c .. of pair i
    const auto finish = [&](int i, float pm, float ps, const f4& po) {
        const int ri = __shfl(row_end >= 0 ? row_end : a.n_rows, i), hi = __shfl(h_end, i);
        if (FORM == kPrefix || (FORM == kOneRow && a.n_own > 0)) {
            if (ri >= a.n_rows) return;
            const int part = (FORM == kPrefix ? a.n_own : 0) + cut;
            const int64_t to = ((int64_t)part * a.n_rows + ri) * a.n_head + hi;
            if (ce == 0) a.part_ms[to] = float2{pm, ps};
            *reinterpret_cast<f4*>(a.part_o + to * kDim + 4 * ce) = po;
        } else {
            const float over = ps == 0.0f ? 0.0f : __fdiv_rn(1.0f, ps);
            attn_store4(a.o, a.n_rows, ri, hi, ce, po * over);
        }
    };
    if constexpr (!SPLIT) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int i = 4 * t + ge;
            finish(i, join_m[we][i], join_s[we][i], *reinterpret_cast<const f4*>(os + i * kPad + 4 * ce));
        }
    } else {  // wave w joins the four waves' pairs 4 w + g
        const int i = 4 * we + ge;
        float M = join_m[0][i];
#pragma unroll
        for (int x = 1; x < 4; ++x) M = fmaxf(M, join_m[x][i]);
        float st = 0.0f;
        f4 ot = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const float f = rescale(join_m[x][i], M);
            st = __fadd_rn(st, __fmul_rn(join_s[x][i], f));
            const f4 ov = *reinterpret_cast<const f4*>(reinterpret_cast<float*>(lds) + (16 * x + i) * kPad + 4 * ce);
#pragma unroll
            for (int e = 0; e < 4; ++e) ot[e] = __fadd_rn(ot[e], __fmul_rn(ov[e], f));
        }
        finish(i, M, st, ot);
    }
    dead_rows();
}

template <class T, int G>
__global__ __launch_bounds__(256) void kv_rows(KvArgs a) {
    rows_of<T, G, 4>(a, blockIdx.x, blockIdx.y);
}

// Workgroups a CU: fp16 stages leave room for four (three: 131 us where four take
// 120, 8 prompts behind a voice), fp32 ones' LDS for three.
template <class T, bool SPLIT, int FORM>
__global__ __launch_bounds__(256, SPLIT ? 2 : sizeof(T) == 2 ? 4 : 3) void kv_tiles(KvArgs a) {
    tiles_of<T, SPLIT, FORM>(a, blockIdx.x, gridDim.x, blockIdx.y);
}

// A step with shared prefixes in one launch: first the workgroups of the
// prefixes' tiles, then those of the rows' own keys (the vector units' or, MX,
// the matrix cores' form): the tiles' products run beside the rows' reads.
// us, in two launches (prefixes + own) and in one: 64 rows behind a prefix of
// 377 keys 15.5 + 9.4, 14.8; 512 rows of up to 64 behind one of 2001 48 + 25,
// 54; 256 fp16 rows of up to 400 behind 8 of 250 to 500 11.6 + 23, 28.  The
// rows have what the tiles leave of the LDS: three workgroups a CU for fp32.
template <class T, int G, int W, bool MX>
__global__ __launch_bounds__(256, 3) void kv_shared(KvArgs a, uint32_t tile_blocks, uint32_t row_blocks) {
    if (blockIdx.x < tile_blocks) {
        const uint32_t n = tile_blocks / a.n_shared;
        tiles_of<T, false, kPrefix>(a, blockIdx.x % n, n, blockIdx.x / n);
    } else {
        const uint32_t b = blockIdx.x - tile_blocks;
        if constexpr (MX) tiles_of<T, true, kOneRow>(a, b % row_blocks, row_blocks, b / row_blocks);
        else rows_of<T, G, W>(a, b % row_blocks, b / row_blocks);
    }
}

// ------------------------------------------------------------------ launches

// How a call's keys are cut: parts of a row's own (0: whole rows, stored by
// the workgroup itself) and of a prefix.  Lengths are the device's: the host knows
// the tables' capacity alone, and cuts for rows as long as that.  Parts that a
// shorter row does not need end at once, but are launched, and its one part goes
// through the workspace and the join: us, tables of 416 / 8196 positions, 64 rows
// of 129 to 383 fp32 keys 29 / 43 (2048: 33, 32768: 87), 63 of them 34 / 42, fp16
// 64 14.8 / 31, 64 of up to 300 behind a prefix of 377 18 / 32; 256 fp16 rows of 64
// to 4001 with four query heads a key head 76 (3968) / 84.
struct Cut {
    int own, shared, min_part;
};

// Row heads from which rows beside prefixes' tiles get a wave each instead of a
// workgroup.  us, a workgroup / a wave: fp32 rows of up to 300 behind a prefix
// of 377, 64 of them 17.6 / 24.3, 128: 23.5 / 25.6, 256: 39.4 / 38.8; fp16 256
// of them 30.7 / 26.1; 512 of 100 behind one of 2001: 142 / 110.  Without tiles
// a workgroup each is as fast or faster at any number (256 fp32 rows of 129 to
// 383: 100 / 107).
constexpr int64_t kWaveUnits = 4096;

int head_chunk(int group) { return group >= 3 ? 4 : group; }

// Whether a key head's query heads are pairs of one tile.  us, vector units /
// matrix cores, 16 fp16 heads, rows of 1000 keys: 2 heads a key head, 64 rows
// 29.3 / 31.7; 4: 64 rows 25.9 / 21.6, 256 67.8 / 62.0; 8: 256 58.0 / 33.0.
bool on_matrix(bool f16, int group) { return f16 && group >= 3; }

// A row's workgroups (or waves) of one part.
int row_units(bool f16, int n_kv, int group) {
    const int G = head_chunk(group);
    return n_kv * (on_matrix(f16, group) ? (group + 15) / 16 : (group + G - 1) / G);
}

Cut cut_of(const cbx_kv_attn& a) {
    Cut c{0, 0, kMinPart};
    if (a.rows->stream) return c;
    const int group = a.n_head / a.cache->n_head;
    const bool f16 = a.cache->type == CBX_KV_F16;
    const int64_t wgs = (int64_t)a.rows->n_rows * row_units(f16, a.cache->n_head, group);
    const int64_t cap = (int64_t)a.streams->max_pages * a.cache->page_size;
    const bool prefixes = a.streams->parent && a.streams->n_prefix > 0;
    const bool tiles = a.rows->tiles && prefixes;
    const int64_t longest = tiles || !prefixes ? cap : 2 * cap;
    // Parts worth a workgroup's start and end, and about as many workgroups as
    // run at a time; of fp32 rows two such rounds where a part is still 256 keys,
    // but none where whole rows fill a round (a join would come on top: 64 rows of
    // 200 keys 19.4 / 24.2).  us: 256 fp16 rows of 64 to 4001 keys, four query heads a key
    // head, parts of 64 keys and more 143, of 512 94; fp32 rows of 64 to 4001
    // keys, one round / two: 8 rows 19.3 / 17.7, 16: 33.8 / 28.9, 32 with four
    // heads a key head 34.6 / 28.8, 64: 57.7 / 38.9, but 16 of these (parts of 125)
    // 21.6 / 23.8, and fp16 32 with four heads 20.4 / 22.8, 16 of 1000 keys with
    // two 15.1 / 17.8
    const bool two = !tiles && !f16 && wgs >= 128 && wgs < 1024;
    c.min_part = two ? (int)std::min<int64_t>(std::max<int64_t>(wgs, 256), 512)
                     : (int)std::min<int64_t>(std::max<int64_t>(wgs / 2, kMinPart), 512);
    int64_t own = ((two ? 2048 : 1024) + wgs - 1) / wgs;
    // a row of many keys in several parts whatever their number (us, parts of
    // 2048 / 1024 / 512 / 256 keys: 256 fp32 rows of 64 to 4001 363 / 355 / 362 /
    // 387); rounded, or rows of just over 1024 come in two halves (64 rows of
    // 1000 97.4 / 92.5)
    own = std::max(own, (longest + 512) / 1024);
    own = std::min(own, std::min<int64_t>(64, (longest + kMinPart - 1) / kMinPart));
    if (tiles) {
        const int64_t t = (int64_t)a.rows->n_tiles * a.cache->n_head;
        const int64_t most = std::min<int64_t>(32, (cap + 63) / 64);
        // prefixes' parts: enough workgroups that rows can run beside them, and
        // not so many that all CUs are theirs first.  us with 768 / 384 / 256
        // workgroups: 512 rows behind 2001 keys 58 / 54 / 71, 256 fp16 rows
        // behind 8 prefixes 30.8 / 28.0 / 27.4; with parts of 32 / 64 keys at
        // least 64 rows behind 377: 16.0 / 14.8
        c.shared = (int)std::min(std::max<int64_t>((384 + t / 2) / t, 1), most);
        // one grid holds both
        c.own = (int)std::min(own, std::max<int64_t>((kMaxKvGrid - t * c.shared) / wgs, 1));
    } else {
        c.own = own > 1 ? (int)own : 0;
    }
    return c;
}

// The step form: the rows' own keys, behind the prefixes' tiles where there are any.
template <class T>
hipError_t launch_step(const KvArgs& a, hipStream_t st) {
    const int G = head_chunk(a.group);
    const bool matrix = on_matrix(sizeof(T) == 2, a.group);
    // beside prefixes' tiles a wave per row and head where those are many: four
    // heads a workgroup, no barrier
    const int64_t units = (int64_t)a.n_rows * row_units(sizeof(T) == 2, a.n_kv, a.group);
    const bool wave = !matrix && a.n_shared && units >= kWaveUnits;
    const unsigned blocks = (unsigned)(wave ? (units + 3) / 4 : units), cuts = (unsigned)max(a.n_own, 1);
    const unsigned tiles = (unsigned)a.n_kv * a.n_tiles * a.n_shared;
    const auto go = [&](auto rows, auto both, auto waves) {
        if (a.n_shared)
            hipLaunchKernelGGL(wave ? waves : both, dim3(tiles + blocks * cuts), dim3(256), 0, st, a, tiles, blocks);
        else
            hipLaunchKernelGGL(rows, dim3(blocks, cuts), dim3(256), 0, st, a);
        return hipGetLastError();
    };
    if (G == 1) return go(kv_rows<T, 1>, kv_shared<T, 1, 4, false>, kv_shared<T, 1, 1, false>);
    if (G == 2) return go(kv_rows<T, 2>, kv_shared<T, 2, 4, false>, kv_shared<T, 2, 1, false>);
    if constexpr (sizeof(T) == 2)
        return go(kv_tiles<T, true, kOneRow>, kv_shared<T, 1, 4, true>, kv_shared<T, 1, 4, true>);
    else
        return go(kv_rows<T, 4>, kv_shared<T, 4, 4, false>, kv_shared<T, 4, 1, false>);
}

template <class T>
hipError_t launch_prompt(const KvArgs& a, hipStream_t st) {
    // few tiles: four workgroups a tile, their waves the same pairs and other keys.
    // Worth it while the workgroups (a.n_tiles counts a tile more per stream than
    // there may be) are about the one or two a CU that fit: us, whole tiles /
    // split, fp32: 1 x 256 rows 17.9 / 13.0, 1 x 384 24.6 / 21.0, 2 x 192 14.9 /
    // 17.0, 4 x 256 20.3 / 40.6; fp16: 1 x 512 21.6 / 14.0, 2 x 256 13.7 / 11.4,
    // 3 x 256 14.4 / 16.2
    const bool split = (int64_t)a.n_tiles * 4 * a.n_kv <= (sizeof(T) == 4 ? 448 : 896);
    const dim3 grid((unsigned)a.n_kv * a.n_tiles * (split ? 4 : 1));
    if (split) hipLaunchKernelGGL((kv_tiles<T, true, kPrompt>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((kv_tiles<T, false, kPrompt>), grid, dim3(256), 0, st, a);
    return hipGetLastError();
}

template <class T>
hipError_t launch(const KvArgs& a, bool step, hipStream_t st) {
    if (!step) return launch_prompt<T>(a, st);
    const hipError_t e = launch_step<T>(a, st);
    if (e != hipSuccess || !a.n_own) return e;
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
    const bool listed = !r.stream || r.tiles;  // prompts' tiles, else found by their numbers
    a.tile_rows = listed ? r.tile_rows : cbx_kv_tile_rows(c.n_head, p.n_head);
    a.n_tiles = listed ? r.n_tiles : r.n_rows / a.tile_rows + s.n_streams;
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
    a.over_group = 65536 / a.group + 1;
    a.scale = c.scale * kLog2e;
    a.o = AttnOut{c.out, c.ld_out, parts, inv, c.n_head};
    const uint64_t n = (uint64_t)(cut.own + cut.shared) * r.n_rows * c.n_head;
    a.part_ms = static_cast<float2*>(c.workspace);
    a.part_o = reinterpret_cast<float*>(static_cast<char*>(c.workspace) + (n * 8 + 255) / 256 * 256);
    a.n_own = cut.own;
    a.n_shared = cut.shared;
    a.min_part = cut.min_part;
    return p.type == CBX_KV_F32 ? launch<float>(a, !r.stream, st) : launch<_Float16>(a, !r.stream, st);
}

}  // namespace cbx
