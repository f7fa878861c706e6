// Which keys each query sees, as one interval a row (the definition is in fa_b200.h), with what the attention kernels
// want to know of 16 and 128 rows and of 128 keys at once.
//
// A thread makes a row: a binary search of its document, a few minima and maxima.  What bounds it is latency: two dependent
// launches (one for up to 128 rows, whose tiles need no order) and the search's chain of loads.  12 bytes a row are written, 1.5 MB at
// 8 rows of 16384 tokens, where a call with 32 documents a row takes 14 us; one row for each of 64 requests 11, most of it the
// host's, which makes a plan, positions and two views.
#include "fa_common.cuh"
#include "sm100_ptx.cuh"
#include <limits.h>

namespace fa {
namespace {

struct RangesArgs {
    int32_t* plan;
    int32_t* positions;
    const int2* rows;
    const int32_t *offsets, *prefixes, *key_lengths, *query_offsets;
    int64_t offsets_sb, prefixes_sb;
    int documents, query_offset, causal, window, B, Nq, Nk;
};

// Saturating, so that no sum of two 32-bit lengths leaves the type.
__device__ __forceinline__ int clamp32(int64_t x) { return (int)(x < -INT_MAX ? -INT_MAX : (x > INT_MAX ? INT_MAX : x)); }

__device__ __forceinline__ int2 row_of(const RangesArgs& a, int b, int i, int64_t t, int& position) {
    position = clamp32(t);
    int64_t first, end;
    if (a.rows) {
        const int2 r = a.rows[(int64_t)b * a.Nq + i];
        first = r.x; end = r.y;
    } else {
        int64_t start = 0;
        int m = 0;
        end = a.Nk;
        if (a.offsets) {
            // the last boundary at or below t
            const int32_t* off = a.offsets + b * a.offsets_sb;
            int lo = -1, hi = a.documents + 1;             // off[lo] <= t < off[hi], as far as they exist
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (off[mid] <= t) lo = mid; else hi = mid;
            }
            if (lo < 0 || lo >= a.documents) { position = 0; return make_int2(0, 0); }
            m = lo;
            start = off[m];
            const int64_t stop = off[m + 1];
            end = end < stop ? end : stop;
            position = clamp32(t - start);
        }
        if (a.key_lengths) { const int64_t n = a.key_lengths[b]; end = end < n ? end : n; }
        first = start;
        if (a.window > 0) {
            const int64_t from = t - a.window + 1;
            first = first > from ? first : from;
            if (!a.causal) { const int64_t to = t + a.window; end = end < to ? end : to; }
        }
        if (a.causal) {
            int64_t to = t + 1;
            if (a.prefixes) {
                const int64_t n = a.prefixes[b * a.prefixes_sb + m];
                if (n > 0 && start + n > to) to = start + n;
            }
            end = end < to ? end : to;
        }
    }
    if (first < 0) first = 0;
    if (end > a.Nk) end = a.Nk;
    return first < end ? make_int2((int)first, (int)end) : make_int2(0, 0);
}

// A block makes the 128 rows of a query tile.
__global__ void __launch_bounds__(128) key_rows_kernel(const RangesArgs a) {
    ptx::grid_launch_dependents();                 // key_orders_kernel or key_tiles_kernel, which waits for this grid's end
    const RangesLayout l = ranges_layout(a.B, a.Nq, a.Nk);
    __shared__ int4 part[4];
    const int tile = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int i = tile * 128 + (int)threadIdx.x;
    const int origin = clamp32((int64_t)a.query_offset + (a.query_offsets ? a.query_offsets[b] : 0));
    int2 r = make_int2(0, 0);
    if (i < a.Nq) {
        int position;
        r = row_of(a, b, i, (int64_t)i + origin, position);
        if (a.positions) a.positions[(int64_t)b * a.Nq + i] = position;
    }
    ((int2*)a.plan)[(int64_t)b * l.nq_pad + i] = r;
    const bool sees = r.x < r.y;
    int4 h;                                        // least first, largest end; largest first, least end
    h.x = sees ? r.x : INT_MAX;
    h.y = sees ? r.y : 0;
    h.z = sees ? r.x : 0;
    h.w = sees ? r.y : INT_MAX;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        h.x = min(h.x, __shfl_xor_sync(0xffffffffu, h.x, off));
        h.y = max(h.y, __shfl_xor_sync(0xffffffffu, h.y, off));
        h.z = max(h.z, __shfl_xor_sync(0xffffffffu, h.z, off));
        h.w = min(h.w, __shfl_xor_sync(0xffffffffu, h.w, off));
        if (off == 8 && (lane & 15) == 0)
            ((int2*)(a.plan + l.q_parts))[(int64_t)b * (l.nq_pad / 16) + i / 16] = h.y > 0 ? make_int2(h.x, h.y) : make_int2(0, 0);
    }
    if (lane == 0) part[warp] = h;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 4; ++w) {
            h.x = min(h.x, part[w].x); h.y = max(h.y, part[w].y); h.z = max(h.z, part[w].z); h.w = min(h.w, part[w].w);
        }
        if (h.y <= 0) h.x = 0;
        ((int4*)(a.plan + l.q_tiles))[(int64_t)b * (l.nq_pad / 128) + tile] = h;
        if (tile == 0) a.plan[l.origin + b] = origin;
        part[0] = h;
    }
    // with one query tile a key tile's list follows from its hull; with several the next launch makes them
    if (l.nq_pad == 128) {
        __syncthreads();
        const int4 whole = part[0];
        int2* k_tiles = (int2*)(a.plan + l.k_tiles) + (int64_t)b * (l.nk_pad / 128);
        int32_t* k_order = a.plan + l.k_order + (int64_t)b * (l.nk_pad / 128);
        for (int j = threadIdx.x; j < l.nk_pad / 128; j += 128) {
            k_tiles[j] = make_int2(0, whole.x < j * 128 + 128 && whole.y > j * 128 ? 1 : 0);
            k_order[j] = j;
        }
        if (threadIdx.x == 0) { a.plan[l.q_order + b] = 0; a.plan[l.p_order + b] = 0; }
    }
}

// Key tiles' lists; the orders as they come.  For many tiles: a warp a key tile, all over the GPU.
__global__ void __launch_bounds__(256) key_tiles_kernel(const RangesArgs a) {
    ptx::grid_dependency_wait();
    const RangesLayout l = ranges_layout(a.B, a.Nq, a.Nk);
    const int j = (int)blockIdx.x * 8 + (int)(threadIdx.x >> 5), b = blockIdx.y, lane = threadIdx.x & 31;
    const int n = l.nq_pad / 128, nk = l.nk_pad / 128, np = (n + 1) / 2;
    for (int i = (int)(blockIdx.x * blockDim.x + threadIdx.x); i < n; i += (int)(gridDim.x * blockDim.x)) {
        a.plan[l.q_order + (int64_t)b * n + i] = n - 1 - i;
        if (i < np) a.plan[l.p_order + (int64_t)b * np + i] = np - 1 - i;
    }
    if (j >= nk) return;
    const int4* q_tiles = (const int4*)(a.plan + l.q_tiles) + (int64_t)b * n;
    int lo = INT_MAX, hi = 0;
    for (int t = lane; t < n; t += 32) {
        const int4 h = q_tiles[t];
        if (h.x < j * 128 + 128 && h.y > j * 128) { lo = min(lo, t); hi = t + 1; }
    }
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if (lane == 0) {
        ((int2*)(a.plan + l.k_tiles))[(int64_t)b * nk + j] = hi > 0 ? make_int2(lo, hi) : make_int2(0, 0);
        a.plan[l.k_order + (int64_t)b * nk + j] = j;
    }
}
// The same for at most kMostOrdered tiles, a block a batch entry, and the orders: a tile's place is the number of tiles that
// meet more others, or as many and come first (later ones first for queries, where a causal mask makes them the longer ones).
__global__ void __launch_bounds__(1024) key_orders_kernel(const RangesArgs a) {
    __shared__ int4 hulls[kMostOrdered];
    __shared__ __align__(16) int cost[3][kMostOrdered];
    const RangesLayout l = ranges_layout(a.B, a.Nq, a.Nk);
    const int b = blockIdx.x, n = l.nq_pad / 128, nk = l.nk_pad / 128, np = (n + 1) / 2;
    for (int i = threadIdx.x; i < 3 * kMostOrdered; i += 1024) (&cost[0][0])[i] = -1;        // (places behind the last tile: no place taken)
    ptx::grid_dependency_wait();
    for (int t = threadIdx.x; t < n; t += 1024) hulls[t] = ((const int4*)(a.plan + l.q_tiles))[(int64_t)b * n + t];
    __syncthreads();
    auto tiles_of = [](int x, int y) { return y > x ? (y + 127) / 128 - x / 128 : 0; };
    static_assert(2 * kMostOrdered == 1024, "half of the threads for the keys, half for the queries");
    if (threadIdx.x < kMostOrdered) {
        // a thread a key tile, which all look at the same query tile
        const int j = threadIdx.x;
        if (j < nk) {
            int lo = INT_MAX, hi = 0;
#pragma unroll 4
            for (int t = 0; t < n; ++t) {
                const int4 h = hulls[t];
                if (h.x < j * 128 + 128 && h.y > j * 128) { lo = min(lo, t); hi = t + 1; }
            }
            const int2 r = hi > 0 ? make_int2(lo, hi) : make_int2(0, 0);
            ((int2*)(a.plan + l.k_tiles))[(int64_t)b * nk + j] = r;
            cost[0][j] = r.y - r.x;
        }
    } else {
        const int t = threadIdx.x - kMostOrdered;
        if (t < n) {
            const int4 h = hulls[t];
            cost[1][t] = tiles_of(h.x, h.y);
            if (t % 2 == 0) {
                const int4 g = t + 1 < n ? hulls[t + 1] : make_int4(0, 0, 0, 0);
                cost[2][t / 2] = h.y <= 0 ? tiles_of(g.x, g.y) : (g.y <= 0 ? tiles_of(h.x, h.y) : tiles_of(min(h.x, g.x), max(h.y, g.y)));
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < nk + n + np; i += 1024) {
        const int o = i < nk ? 0 : (i < nk + n ? 1 : 2), count = o == 0 ? nk : (o == 1 ? n : np), me = i - (o == 0 ? 0 : (o == 1 ? nk : nk + n));
        const int mine = cost[o][me];
        int place = 0;
        for (int e = 0; e < count; e += 4) {
            const int4 c = *reinterpret_cast<const int4*>(&cost[o][e]);
            auto ahead = [&](int x, int at) { return x > mine || (x == mine && (o == 0 ? at < me : at > me)); };
            place += ahead(c.x, e) + ahead(c.y, e + 1) + ahead(c.z, e + 2) + ahead(c.w, e + 3);
        }
        const int64_t base = o == 0 ? l.k_order + (int64_t)b * nk : (o == 1 ? l.q_order + (int64_t)b * n : l.p_order + (int64_t)b * np);
        a.plan[base + place] = me;
    }
}

}  // namespace
}  // namespace fa

using namespace fa;

extern "C" {

size_t fa_b200_key_ranges_bytes(int B, int Nq, int Nk) {
    if (B < 0 || Nq < 0 || Nk < 0) return 0;
    return (size_t)ranges_layout(B, Nq, Nk).total * sizeof(int32_t);
}

int fa_b200_key_ranges(const fa_b200_ranges_params* p) {
    if (!p) { set_error("params is null"); return FA_EINVAL; }
    if (p->struct_bytes != sizeof(fa_b200_ranges_params)) {
        set_error("struct_bytes %zu does not match this library's fa_b200_ranges_params (%zu bytes)", p->struct_bytes, sizeof(fa_b200_ranges_params));
        return FA_EINVAL;
    }
    if (p->B < 0 || p->Nq < 0 || p->Nk < 0) { set_error("key_ranges: negative size"); return FA_EINVAL; }
    if (p->Nq > INT_MAX - 256 || p->Nk > INT_MAX - 256) { set_error("key_ranges: lengths must stay below 2^31 - 256"); return FA_EUNSUPPORTED; }
    if (p->B > 65535) { set_error("key_ranges: batch must be below 65536"); return FA_EUNSUPPORTED; }
    if (p->window < 0) { set_error("key_ranges: window %d is negative", p->window); return FA_EINVAL; }
    if (p->n_documents < 0 || (p->document_offsets && p->n_documents == 0)) { set_error("key_ranges: document_offsets without documents"); return FA_EINVAL; }
    if (p->prefix_lengths && (!p->causal || p->window > 0)) { set_error("key_ranges: prefixes are defined for causal ranges without a window"); return FA_EINVAL; }
    if (p->B == 0 || p->Nq == 0) return FA_OK;
    if (!p->plan) { set_error("key_ranges: plan is null"); return FA_EINVAL; }
    if (((uintptr_t)p->plan & 15u) != 0 || ((uintptr_t)p->rows & 7u) != 0) { set_error("key_ranges: plan must be 16-byte aligned, rows 8"); return FA_EALIGN; }
    if (p->plan_bytes < fa_b200_key_ranges_bytes(p->B, p->Nq, p->Nk)) {
        set_error("key_ranges: plan holds %zu bytes, %zu are needed", p->plan_bytes, fa_b200_key_ranges_bytes(p->B, p->Nq, p->Nk));
        return FA_EWORKSPACE;
    }
    GuardDevice g(p->device);
    if (!g.ok) { set_error("cudaSetDevice(%d) failed", p->device); return FA_ECUDA; }
    RangesArgs a;
    a.plan = (int32_t*)p->plan; a.positions = p->positions; a.rows = (const int2*)p->rows;
    a.offsets = p->document_offsets; a.prefixes = p->prefix_lengths; a.key_lengths = p->key_lengths; a.query_offsets = p->query_offsets;
    a.offsets_sb = p->offsets_stride_b; a.prefixes_sb = p->prefix_stride_b;
    a.documents = p->n_documents; a.query_offset = p->query_offset; a.causal = p->causal; a.window = p->window;
    a.B = p->B; a.Nq = p->Nq; a.Nk = p->Nk;
    const RangesLayout l = ranges_layout(p->B, p->Nq, p->Nk);
    cudaStream_t st = (cudaStream_t)p->stream;
    key_rows_kernel<<<dim3((unsigned)(l.nq_pad / 128), (unsigned)p->B), 128, 0, st>>>(a);
    FA_CUDA_CHECK(cudaGetLastError());
    if (l.nq_pad > 128 && l.nk_pad > 0) {
        const bool ordered = l.nq_pad / 128 <= kMostOrdered && l.nk_pad / 128 <= kMostOrdered;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = ordered ? dim3((unsigned)p->B) : dim3((unsigned)((l.nk_pad / 128 + 7) / 8), (unsigned)p->B);
        cfg.blockDim = dim3(ordered ? 1024 : 256);
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        FA_CUDA_CHECK(cudaLaunchKernelEx(&cfg, ordered ? key_orders_kernel : key_tiles_kernel, a));
    }
    return FA_OK;
}

}  // extern "C"
