// cbx_kv_plan.hip -- page tables, slot maps and row tiles of a paged cache's
// call from the streams' lengths (cbx_kv_build, include/cbx_kv.h).
//
// With c_i the rows granted to stream i and t_i the pages taken for them,
//   row_start[i]  = sum over j < i of c_j
//   page_start[i] = sum over j < i of t_j
// the page of stream i's own index held_i + j is free_pages[F - 1 -
// (page_start[i] + j)], F the free count, and row row_start[i] + x is that of
// its own position len_i + x.  So a call is a few sums over the streams, then
// one entry per row, page and tile, each found from the sums alone.
//
// One workgroup makes the sums (thread t: streams PER t ..), and in the step
// form, or where the rows are few, all entries too; else a second launch over
// all CUs writes the rows and pages, each thread finding its stream by
// bisection of the sums.  Bound by its chain of dependent loads and the
// launches: the bytes (12 a row, 8 a page) take less.  us a call: a step of 64
// streams 7.6, 64 prompts of 129 to 383 rows 12.3, 2048 of up to 383 18.2 (12.0
// and 7.1 the two kernels), of which 5 to 6 are a launch's own.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "cbx_internal.h"

namespace cbx {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;

struct PlanArgs {
    cbx_kv_streams s;
    cbx_kv_rows r;
    int32_t shift;  // page_size = 1 << shift
    const int32_t* n_new;
    const int32_t* state;
    const int32_t* release;
    int32_t* len_out;
    int32_t* n_free_out;
};

__device__ __forceinline__ int pages_of(const PlanArgs& a, int len) {
    return (int)(((int64_t)len + (1 << a.shift) - 1) >> a.shift);
}

// A stream's prefix, and how much of it the stream shares (0: none).
__device__ __forceinline__ int prefix_of(const PlanArgs& a, int i, int& len) {
    len = 0;
    if (!a.s.parent || i < a.s.n_prefix) return -1;
    const int p = a.s.parent[i];
    if (p < 0 || p >= a.s.n_prefix) return -1;
    len = min(max(a.s.prefix_len[i], 0), a.s.max_pages << a.shift);
    return p;
}

__device__ __forceinline__ int slot_of(const PlanArgs& a, int page, int off) {
    return page >= 0 && page < a.s.n_pages ? (page << a.shift) + (off & ((1 << a.shift) - 1)) : -1;
}

// Inclusive sum over the workgroup's threads of v; `sums` holds kPlanWaves
// values, free again when the next call's threads have passed its barrier (two
// arrays in turn).  total: the sum over all threads.
__device__ int64_t block_scan(int64_t v, int64_t* sums, int64_t& total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t x = __shfl_up(v, o);
        if (lane >= o) v += x;
    }
    if (lane == 63) sums[w] = v;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < kPlanWaves; ++i) {
        const int64_t x = sums[i];
        if (i < w) before += x;
        total += x;
    }
    return v + before;
}

// The largest i < n with start[i] <= x (start[0] = 0, non-decreasing, x below
// start[n]): the stream that holds row (page) x.
__device__ __forceinline__ int holder(const int32_t* start, int lo, int hi, int x) {
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Prompt form: row x's entries, and the x-th page taken (first the pages held
// before the call, from the sums).
__device__ __forceinline__ void fill_row(const PlanArgs& a, int x, int rows, int n_free) {
    if (x >= rows) {
        a.r.stream[x] = a.r.position[x] = a.r.slot[x] = -1;
        return;
    }
    const int i = holder(a.r.row_start, 0, a.s.n_streams, x);
    const int r0 = a.r.row_start[i], had = a.len_out[i] - (a.r.row_start[i + 1] - r0);
    const int off = had + x - r0, held = pages_of(a, had), j = off >> a.shift;
    const int page = j < held ? a.s.tables[(int64_t)i * a.s.max_pages + j]
                              : a.s.free_pages[n_free - 1 - (a.r.page_start[i] + j - held)];
    int plen;
    prefix_of(a, i, plen);
    a.r.stream[x] = i;
    a.r.position[x] = plen + off;
    a.r.slot[x] = slot_of(a, page, off);
}

__device__ __forceinline__ void fill_page(const PlanArgs& a, int x, int n_free) {
    const int i = holder(a.r.page_start, 0, a.s.n_streams, x);
    const int had = a.len_out[i] - (a.r.row_start[i + 1] - a.r.row_start[i]);
    a.s.tables[(int64_t)i * a.s.max_pages + pages_of(a, had) + x - a.r.page_start[i]] =
        a.s.free_pages[n_free - 1 - x];
}

// The sums and everything that is per stream.  FILL: the prompt form's rows
// and pages too.
template <int PER, bool STEP, bool FILL>
__global__ __launch_bounds__(kPlanThreads) void kv_plan(PlanArgs a) {
    __shared__ int64_t sums[2][kPlanWaves];
    extern __shared__ int32_t lds[];  // step form with tiles: [n_prefix] then [n_streams]
    const int tid = threadIdx.x, lane = tid & 63, n = a.s.n_streams;
    const int cap = a.s.max_pages << a.shift;
    int len[PER], want[PER], back[PER];
    int asked = 0, n_back = 0;
    int n_free = min(max(a.s.n_free[0], 0), a.s.n_pages);
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        const int i = tid * PER + u;
        len[u] = want[u] = back[u] = 0;
        if (i >= n) continue;
        const int l = a.s.len[i];
        const bool ok = l >= 0 && l <= cap;
        len[u] = l;
        int w = a.n_new ? max(a.n_new[i], 0) : 1;
        if (a.state && a.state[i] != CBX_DECODE_RUNNING) w = 0;
        if (STEP) w = min(w, 1);
        asked += w > 0;
        if (ok && a.release && a.release[i] != 0) {
            back[u] = pages_of(a, l);
            len[u] = 0;
        }
        want[u] = ok && w <= cap - len[u] ? w : 0;
        n_back += back[u];
    }
    int64_t total;
    int ph = 0;
    const auto scan = [&](int64_t v) {
        const int64_t x = block_scan(v, sums[ph], total);
        ph ^= 1;
        return x;
    };
    if (a.release) {  // the pages given back, a wave copying a stream's at a time
        int64_t at = scan(n_back) - n_back;  // lengths may claim any number of pages
        const int64_t all = total;
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            for (uint64_t left = __ballot(back[u] > 0); left; left &= left - 1) {
                const int from = (int)__builtin_ctzll(left);
                const int k = __shfl(back[u], from);
                const int64_t to = n_free + __shfl(at, from);
                const int64_t src = (int64_t)((tid & ~63) + from) * PER + u;
                for (int j = lane; j < k && to + j < a.s.n_pages; j += 64)
                    a.s.free_pages[to + j] = a.s.tables[src * a.s.max_pages + j];
            }
            at += back[u];
        }
        n_free = (int)min((int64_t)a.s.n_pages, n_free + all);
        __syncthreads();  // read as free pages, and the tables written, from here on
    }
    if (!STEP) {  // rows asked up to and with a stream's
        int64_t sum = 0;
#pragma unroll
        for (int u = 0; u < PER; ++u) sum += want[u];
        int64_t at = scan(sum) - sum;
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            at += want[u];
            if (at > a.r.n_rows) want[u] = 0;
        }
    }
    int take[PER];
    {
        int64_t sum = 0;
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            take[u] = want[u] ? pages_of(a, len[u] + want[u]) - pages_of(a, len[u]) : 0;
            sum += take[u];
        }
        int64_t at = scan(sum) - sum;
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            at += take[u];
            if (take[u] && at > n_free) want[u] = take[u] = 0;
        }
    }
    // rows and pages before each stream in one sum: both stay below 2^31
    int64_t both = 0;
    int refused = asked;
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        both += ((int64_t)take[u] << 32) + want[u];
        refused -= want[u] > 0;
    }
    const int64_t before = scan(both) - both;
    const int rows = (int)(total & 0x7fffffff), pages = (int)(total >> 32);
    const int r0 = (int)(before & 0x7fffffff), p0 = (int)(before >> 32);
    int n_tile = 0;
    const int T = a.r.tile_rows;
    if (!STEP && a.r.tiles) {
#pragma unroll
        for (int u = 0; u < PER; ++u) n_tile += (want[u] + T - 1) / T;
    }
    const int64_t more = scan(((int64_t)refused << 32) + n_tile);
    int t0 = (int)(more & 0x7fffffff) - n_tile, tiles = (int)(total & 0x7fffffff);
    if (tid == 0) {
        a.n_free_out[0] = n_free - pages;
        a.r.row_start[n] = rows;
        a.r.page_start[n] = pages;
        a.r.counts[0] = rows;
        a.r.counts[2] = pages;
        a.r.counts[3] = (int)(total >> 32);
        if (!STEP || !a.r.tiles) a.r.counts[1] = tiles;
    }
    int4* const tile = reinterpret_cast<int4*>(a.r.tiles);
    int r = r0, p = p0;
    int key[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        const int i = tid * PER + u;
        key[u] = -1;
        if (i >= n) continue;
        a.r.row_start[i] = r;
        a.r.page_start[i] = p;
        a.len_out[i] = len[u] + want[u];
        if constexpr (STEP) {
            int plen, pos = -1, slot = -1;
            const int pre = prefix_of(a, i, plen);
            if (want[u]) {
                const int64_t at = (int64_t)i * a.s.max_pages + (len[u] >> a.shift);
                const int page = take[u] ? a.s.free_pages[n_free - 1 - p] : a.s.tables[at];
                if (take[u]) a.s.tables[at] = page;
                pos = plen + len[u];
                slot = slot_of(a, page, len[u]);
                if (plen > 0) key[u] = pre;
            }
            a.r.position[i] = pos;
            a.r.slot[i] = slot;
        } else if (tile) {
            int plen;
            prefix_of(a, i, plen);
            for (int f = 0; f < want[u]; f += T) {
                const int c = min(T, want[u] - f);
                tile[t0++] = make_int4(i, r + f, c, plen + len[u] + f + c);
            }
        }
        r += want[u];
        p += take[u];
    }
    if constexpr (!STEP) {
        for (int t = tiles + tid; tile && t < a.r.n_tiles; t += kPlanThreads)
            tile[t] = make_int4(-1, 0, 0, 0);
        if constexpr (FILL) {
            __syncthreads();
            for (int x = tid; x < pages; x += kPlanThreads) fill_page(a, x, n_free);
            for (int x = tid; x < a.r.n_rows; x += kPlanThreads) fill_row(a, x, rows, n_free);
        }
        return;
    }
    if (!tile) return;
    // Step form: the rows with a prefix in order of their prefix, streams in
    // order within one.  Counted per prefix, then placed by one wave, 64
    // streams at a time, each after those of its prefix before it.
    int* const at = lds;
    int* const keys = lds + a.s.n_prefix;
    for (int i = tid; i < a.s.n_prefix; i += kPlanThreads) at[i] = 0;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        const int i = tid * PER + u;
        if (i >= n) continue;
        keys[i] = key[u];
        if (key[u] >= 0) atomicAdd(&at[key[u]], 1);
    }
    __syncthreads();
    const int per = (a.s.n_prefix + kPlanThreads - 1) / kPlanThreads;
    const int q0 = min(tid * per, a.s.n_prefix), q1 = min(q0 + per, a.s.n_prefix);
    int64_t sum = 0;  // tiles and rows of this thread's prefixes
    for (int q = q0; q < q1; ++q) sum += ((int64_t)((at[q] + T - 1) / T) << 32) + at[q];
    const int64_t first = scan(sum) - sum;
    const int grouped = (int)(total & 0x7fffffff);
    tiles = (int)(total >> 32);
    int f = (int)(first & 0x7fffffff), t = (int)(first >> 32);
    for (int q = q0; q < q1; ++q) {
        const int c = at[q];
        for (int x = 0; x < c; x += T) tile[t++] = make_int4(q, f + x, min(T, c - x), 0);
        at[q] = f;
        f += c;
    }
    for (int x = tiles + tid; x < a.r.n_tiles; x += kPlanThreads) tile[x] = make_int4(-1, 0, 0, 0);
    for (int x = grouped + tid; x < n; x += kPlanThreads) a.r.order[x] = -1;
    if (tid == 0) a.r.counts[1] = tiles;
    __syncthreads();
    if (tid < 64) {
        for (int i0 = 0; i0 < n; i0 += 64) {
            const int k = i0 + lane < n ? keys[i0 + lane] : -1;
            uint64_t same = __ballot(k >= 0);  // the lanes of this lane's prefix
            if (!same) continue;
#pragma unroll
            for (int bit = 0; bit < 14; ++bit) {
                const uint64_t on = __ballot((k >> bit) & 1);
                same &= (k >> bit) & 1 ? on : ~on;
            }
            const int rank = __popcll(same & ((1ull << lane) - 1));
            const int place = k >= 0 ? at[k] : 0;
            // every lane has read its place before the first of a prefix moves
            // it on, and that is seen by the next 64
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
            __builtin_amdgcn_wave_barrier();
            if (k >= 0) a.r.order[place + rank] = i0 + lane;
            if (k >= 0 && rank == 0) at[k] = place + __popcll(same);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
            __builtin_amdgcn_wave_barrier();
        }
    }
    __syncthreads();
    // a tile's keys: the longest prefix of its rows, a wave per tile
    for (int x = tid >> 6; x < tiles; x += kPlanWaves) {
        const int4 d = tile[x];
        int most = 0;
        for (int c = lane; c < d.z; c += 64) {
            int plen;
            prefix_of(a, a.r.order[d.y + c], plen);
            most = max(most, plen);
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) most = max(most, __shfl_xor(most, o));
        if (lane == 0) tile[x].w = most;
    }
}

// The prompt form's rows and pages over all CUs.
constexpr int kFillThreads = 256;
__global__ __launch_bounds__(kFillThreads) void kv_fill(PlanArgs a) {
    const int n = a.s.n_streams;
    const int rows = a.r.row_start[n], pages = a.r.page_start[n];
    const int n_free = a.n_free_out[0] + pages;
    const int x0 = blockIdx.x * kFillThreads + threadIdx.x, step = gridDim.x * kFillThreads;
    for (int64_t x = x0; x < pages; x += step) fill_page(a, (int)x, n_free);
    for (int64_t x = x0; x < a.r.n_rows; x += step) fill_row(a, (int)x, rows, n_free);
}

template <int PER, bool STEP, bool FILL>
hipError_t launch(const PlanArgs& a, hipStream_t st) {
    const size_t lds = STEP && a.r.tiles ? 4 * ((size_t)a.s.n_prefix + a.s.n_streams) : 0;
    if (lds > 65536) {
        const hipError_t e =
            hipFuncSetAttribute(reinterpret_cast<const void*>(kv_plan<PER, STEP, FILL>),
                                hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((kv_plan<PER, STEP, FILL>), dim3(1), dim3(kPlanThreads), lds, st, a);
    return hipGetLastError();
}

template <bool STEP, bool FILL>
hipError_t launch_per(const PlanArgs& a, hipStream_t st) {
    if (a.s.n_streams <= kPlanThreads) return launch<1, STEP, FILL>(a, st);
    if (a.s.n_streams <= 4 * kPlanThreads) return launch<4, STEP, FILL>(a, st);
    return launch<16, STEP, FILL>(a, st);
}

}  // namespace

// Rows up to which one workgroup writes the prompt form's entries itself.  us a
// call, itself / by kv_fill, prompts of 256 rows: 8 of them 8.0 / 11.9, 16: 10.1 /
// 12.0, 32: 15.6 / 12.0, 64: 28.4 / 12.0.
constexpr int kFillInPlan = 4096;

hipError_t launch_kv_plan(const cbx_kv_plan& p, hipStream_t st) {
    PlanArgs a{*p.streams, *p.rows, __builtin_ctz((unsigned)p.page_size), p.n_new, p.state, p.release,
               p.len_out ? p.len_out : p.streams->len,
               p.len_out ? p.n_free_out : p.streams->n_free};
    if (!a.r.stream) return launch_per<true, false>(a, st);
    if (a.r.n_rows <= kFillInPlan) return launch_per<false, true>(a, st);
    const hipError_t e = launch_per<false, false>(a, st);
    if (e != hipSuccess) return e;
    const int wgs = min((a.r.n_rows + kFillThreads - 1) / kFillThreads, 4096);
    hipLaunchKernelGGL(kv_fill, dim3((unsigned)wgs), dim3(kFillThreads), 0, st, a);
    return hipGetLastError();
}

}  // namespace cbx
