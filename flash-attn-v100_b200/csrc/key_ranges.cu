// Which keys each query sees, as one interval a row (the definition is in fa_b200.h), with what the attention kernels
// want to know of 16 and 128 rows and of 128 keys at once.
//
// A thread makes a row: a binary search of its document, a few minima and maxima.  What bounds it is latency, two
// dependent launches and the search's chain of loads: 12 bytes a row are written, 1.5 MB at 8 rows of 16384 tokens.
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
    ptx::grid_launch_dependents();                 // key_tiles_kernel, which waits for this grid's end
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
    h.z = i < a.Nq ? (sees ? r.x : INT_MAX) : 0;
    h.w = i < a.Nq ? (sees ? r.y : 0) : INT_MAX;
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
        for (int j = threadIdx.x; j < l.nk_pad / 128; j += 128)
            k_tiles[j] = make_int2(0, whole.x < j * 128 + 128 && whole.y > j * 128 ? 1 : 0);
    }
}

// A warp makes a key tile's list: the first and the last query tile whose hull meets it.
__global__ void __launch_bounds__(256) key_tiles_kernel(const RangesArgs a) {
    ptx::grid_dependency_wait();
    const RangesLayout l = ranges_layout(a.B, a.Nq, a.Nk);
    const int j = (int)blockIdx.x * 8 + (int)(threadIdx.x >> 5), b = blockIdx.y, lane = threadIdx.x & 31;
    if (j >= l.nk_pad / 128) return;
    const int n = l.nq_pad / 128;
    const int4* q_tiles = (const int4*)(a.plan + l.q_tiles) + (int64_t)b * n;
    int lo = INT_MAX, hi = 0;
    for (int t = lane; t < n; t += 32) {
        const int4 h = q_tiles[t];
        if (h.x < j * 128 + 128 && h.y > j * 128) { lo = min(lo, t); hi = t + 1; }
    }
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, off));
        hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, off));
    }
    if (lane == 0) ((int2*)(a.plan + l.k_tiles))[(int64_t)b * (l.nk_pad / 128) + j] = hi > 0 ? make_int2(lo, hi) : make_int2(0, 0);
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
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)((l.nk_pad / 128 + 7) / 8), (unsigned)p->B);
        cfg.blockDim = dim3(256);
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        FA_CUDA_CHECK(cudaLaunchKernelEx(&cfg, key_tiles_kernel, a));
    }
    return FA_OK;
}

}  // extern "C"
