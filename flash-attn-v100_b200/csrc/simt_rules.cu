// CUDA-core attention under rules (fa_b200_rules): fp32 calls, in exact fp32 FMA arithmetic, and 16-bit ones whose head size or
// addresses the tensor-core kernels do not take.  A 32-row tile stays in shared memory, 64-row tiles of the other side go by:
//
//   forward   u = scale q.k, x = cap tanh(u / cap) - slope |i - j|, softmax over the row's range with a running maximum, O += P V
//   backward  P = exp(x - lse), dS = P (dP - delta) dx/du; dQ = scale dS K with queries in place (MODE 1), dV = P^T dO and
//             dK = scale dS^T Q with keys in place (MODE 0): every sum has one owner and one order
//
// What bounds large calls is the FMA pipe, and beside it shared memory: a thread takes 4 x 4 scores, or 4 rows by DC / 16 columns
// of a result, two to a packed FMA, and reads 16 bytes at a time (rows DC + 4 floats apart: no bank conflicts).  Scores keep sums
// of even and odd columns, added at the end; results are pairs of columns, with P or dS in both halves.  Small calls have few
// tiles, which is why these have 32 rows, and wait for memory, which is why tiles of fp32 come by asynchronous copies, the next
// ones beside the products.  Forward and backward of B2 N500 H4 D64 with five documents 31 + 73 us, which
// scalar tiles of 64 rows took 61 + 157 for; B4 N4096 H16 D64 causal 34 and 24 TFLOP/s of the 72 that the pipe has, held back by
// the reads beside it (lanes set so that neighbours share addresses: 5 %; more warps an SM: nothing).
//
// Rows of K and V outside the hull of a query tile's ranges are read as zeros, so that memory nobody sees may hold anything.
#include "fa_common.cuh"
#include "sm100_ptx.cuh"
#include <math.h>

namespace fa {
namespace {

using namespace ptx;

constexpr int NT = 128;            // threads: 8 groups of four rows x 16
constexpr int BX = 32;             // rows of the tile that stays
constexpr int BY = 64;             // rows of the tiles that go by
constexpr int SLD = BY + 4;        // row pitch of P and dS

struct RuledArgs {
    fa_b200_tensor q, k, v, o, o_lo, d_o, dq, dk, dv;
    float* lse;
    const float* delta;
    int B, Nq, Nk, H, Hkv, D;
    int pieces;                    // fp32, 16-byte addresses and strides, D a multiple of 4
    float scale;
    Rules rules;
};

// A warp has two groups of four rows, lane by lane: neighbours then share a column's address, lanes two apart a row's.
__device__ __forceinline__ int group_of_four() { return (threadIdx.x >> 5) * 2 + (threadIdx.x & 1); }
__device__ __forceinline__ int column_of_group() { return (threadIdx.x & 31) >> 1; }

struct RowRule { int first, end, position; };
__device__ __forceinline__ RowRule row_rule(const RuledArgs& a, int b, int i) {
    RowRule r = {0, 0, 0};
    if (i < a.Nq) {
        const int2 x = a.rules.rows[b * a.rules.rows_b + i];
        r.first = x.x; r.end = x.y;
        r.position = i + a.rules.origin[b * a.rules.origin_b];
    }
    return r;
}
// Keys that rows of a tile of N queries see ((0, 0): none).
template <int N>
__device__ __forceinline__ int2 hull_of(const RuledArgs& a, int b, int tile) {
    const int2* parts = a.rules.q_parts + b * a.rules.q_parts_b + tile * (N / 16);
    int2 r = make_int2(0x7fffffff, 0);
#pragma unroll
    for (int e = 0; e < N / 16; ++e) {
        const int2 h = parts[e];
        if (h.y > 0) { r.x = min(r.x, h.x); r.y = max(r.y, h.y); }
    }
    return r.y > 0 ? make_int2(max(r.x, 0), min(r.y, a.Nk)) : make_int2(0, 0);
}
// x of a score u = scale q.k, and the derivative of x by u
__device__ __forceinline__ float ruled_score(float cap, float slope, float u, int position, int key, float& dx) {
    dx = 1.f;
    if (cap > 0.f) {
        const float t = tanhf(u / cap);
        u = cap * t;
        dx = 1.f - t * t;
    }
    return u - slope * fabsf((float)(position - key));         // (floats of their own would round positions from 2^24 on)
}

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// ROWS rows from row0 on; rows outside [lo, hi) and columns from D on are zeros.  There after cp_async_wait and a barrier.
template <typename T, int DC, int ROWS>
__device__ __forceinline__ void copy_rows(float* dst, const T* base, int64_t stride, int row0, int lo, int hi, int D, bool pieces) {
    constexpr int P = DC + 4;
    if (sizeof(T) == 4 && pieces) {
#pragma unroll 4
        for (int e = threadIdx.x; e < ROWS * (DC / 4); e += NT) {
            const int r = e / (DC / 4), c = e % (DC / 4) * 4, row = row0 + r;
            const bool there = row >= lo && row < hi && c < D;
            cp_async_16(smem_u32(dst + r * P + c), there ? base + row * stride + c : base, there ? 16 : 0);
        }
    } else {
#pragma unroll 4
        for (int e = threadIdx.x; e < ROWS * DC; e += NT) {
            const int r = e / DC, c = e % DC, row = row0 + r;
            dst[r * P + c] = row >= lo && row < hi && c < D ? to_f32<T>(base[row * stride + c]) : 0.f;
        }
    }
}

// acc[r][c] += x row (4 ty + r) . y row (tx + 16 c), sums of even and odd columns
template <int DC>
__device__ __forceinline__ void dots(uint64_t (&acc)[4][4], const float* x, const float* y, int ty, int tx) {
    constexpr int P = DC + 4;
#pragma unroll 4
    for (int d = 0; d < DC; d += 4) {
        ulonglong2 xs[4], ys[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) xs[r] = *reinterpret_cast<const ulonglong2*>(x + (ty * 4 + r) * P + d);
#pragma unroll
        for (int c = 0; c < 4; ++c) ys[c] = *reinterpret_cast<const ulonglong2*>(y + (tx + 16 * c) * P + d);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                acc[r][c] = f2_fma(xs[r].x, ys[c].x, acc[r][c]);
                acc[r][c] = f2_fma(xs[r].y, ys[c].y, acc[r][c]);
            }
    }
}

// A thread's columns of a result: pairs 0, 1 from 4 tx on, pairs 2, 3 from 64 + 4 tx (DC = 32: one pair from 2 tx on).
template <int DC>
__device__ __forceinline__ int column_of(int tx, int pair) { return DC == 32 ? tx * 2 : (pair >> 1) * 64 + tx * 4 + (pair & 1) * 2; }
// acc[r][pair] += sum over y of s[4 ty + r][y] * rows[y][columns]
template <int DC>
__device__ __forceinline__ void weigh(uint64_t (&acc)[4][DC / 32], const float* s, const float* rows, int ty, int tx) {
    constexpr int P = DC + 4, N = DC / 32;
#pragma unroll 2
    for (int y = 0; y < BY; y += 4) {
        float w[4][4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float4 x = *reinterpret_cast<const float4*>(s + (ty * 4 + r) * SLD + y);
            w[r][0] = x.x; w[r][1] = x.y; w[r][2] = x.z; w[r][3] = x.w;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            uint64_t v[N];
            if constexpr (N == 1) v[0] = *reinterpret_cast<const uint64_t*>(rows + (y + e) * P + tx * 2);
            else {
#pragma unroll
                for (int g = 0; g < N; g += 2) {
                    const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(rows + (y + e) * P + g * 32 + tx * 4);
                    v[g] = x.x; v[g + 1] = x.y;
                }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint64_t both = f2_pack(w[r][e], w[r][e]);
#pragma unroll
                for (int g = 0; g < N; ++g) acc[r][g] = f2_fma(both, v[g], acc[r][g]);
            }
        }
    }
}
__device__ __forceinline__ float f2_sum(uint64_t x) {
    float lo, hi;
    f2_unpack(x, lo, hi);
    return lo + hi;
}

// A tile's 32 queries; the rows of a half-warp (16 threads, 64 keys) are its own, so maxima, sums and P stay within it.
template <typename T, int DC>
__global__ void __launch_bounds__(NT, DC == 128 ? 2 : 4) ruled_fwd_kernel(const RuledArgs a) {
    constexpr int P = DC + 4, N = DC / 32;
    extern __shared__ __align__(16) float smem[];
    float* Qs = smem;
    float* Ks = Qs + BX * P;
    float* Vs = Ks + BY * P;
    float* Ps = Vs + BY * P;
    const int ty = group_of_four(), tx = column_of_group();
    const int tile = gridDim.x - 1 - blockIdx.x, h = blockIdx.y, b = blockIdx.z, hk = h / (a.H / a.Hkv), m0 = tile * BX;    // (long rows first)
    const T* q = (const T*)a.q.ptr + b * a.q.stride_b + h * a.q.stride_h;
    const T* k = (const T*)a.k.ptr + b * a.k.stride_b + hk * a.k.stride_h;
    const T* v = (const T*)a.v.ptr + b * a.v.stride_b + hk * a.v.stride_h;
    const int2 hull = hull_of<BX>(a, b, tile);
    int n0 = hull.x / BY * BY;
    copy_rows<T, DC, BX>(Qs, q, a.q.stride_n, m0, 0, a.Nq, a.D, a.pieces);
    if (n0 < hull.y) copy_rows<T, DC, BY>(Ks, k, a.k.stride_n, n0, hull.x, hull.y, a.D, a.pieces);
    const float slope = a.rules.slopes ? a.rules.slopes[h] : 0.f;
    RowRule rule[4];
    float m[4], l[4];
    uint64_t acc[4][N];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        rule[r] = row_rule(a, b, m0 + ty * 4 + r);
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int g = 0; g < N; ++g) acc[r][g] = 0;
    }

    for (; n0 < hull.y; n0 += BY) {
        cp_async_wait();
        __syncthreads();                       // K is there, V given back
        copy_rows<T, DC, BY>(Vs, v, a.v.stride_n, n0, hull.x, hull.y, a.D, a.pieces);
        uint64_t s2[4][4] = {};
        dots<DC>(s2, Qs, Ks, ty, tx);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float x[4], top = m[r];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int j = n0 + tx + 16 * c;
                float dx;
                x[c] = ruled_score(a.rules.cap, slope, f2_sum(s2[r][c]) * a.scale, rule[r].position, j, dx);
                if (j < rule[r].first || j >= rule[r].end) x[c] = -INFINITY;
                top = fmaxf(top, x[c]);
            }
#pragma unroll
            for (int w = 2; w < 32; w *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
            const float use = top == -INFINITY ? 0.f : top, alpha = expf(m[r] - use);
            m[r] = top;
            l[r] *= alpha;
            const uint64_t alpha2 = f2_pack(alpha, alpha);
#pragma unroll
            for (int g = 0; g < N; ++g) acc[r][g] = f2_mul(acc[r][g], alpha2);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float p = expf(x[c] - use);
                l[r] += p;
                Ps[(ty * 4 + r) * SLD + tx + 16 * c] = p;
            }
        }
        cp_async_wait();
        __syncthreads();                       // V is there, K given back, P written
        if (n0 + BY < hull.y) copy_rows<T, DC, BY>(Ks, k, a.k.stride_n, n0 + BY, hull.x, hull.y, a.D, a.pieces);
        weigh<DC>(acc, Ps, Vs, ty, tx);
    }
    cp_async_wait();
#pragma unroll
    for (int r = 0; r < 4; ++r) {
#pragma unroll
        for (int w = 2; w < 32; w *= 2) l[r] += __shfl_xor_sync(0xffffffffu, l[r], w);
        const int i = m0 + ty * 4 + r;
        if (i >= a.Nq) continue;
        const float inv = l[r] == 0.f ? 0.f : 1.f / l[r];          // (a row that sees nothing)
        T* o = (T*)a.o.ptr + b * a.o.stride_b + i * a.o.stride_n + h * a.o.stride_h;
        T* lo = a.o_lo.ptr ? (T*)a.o_lo.ptr + b * a.o_lo.stride_b + i * a.o_lo.stride_n + h * a.o_lo.stride_h : nullptr;
#pragma unroll
        for (int g = 0; g < N; ++g) {
            float x[2];
            f2_unpack(acc[r][g], x[0], x[1]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int col = column_of<DC>(tx, g) + e;
                if (col >= a.D) continue;
                const T hi = from_f32<T>(x[e] * inv);
                o[col] = hi;
                if (lo) lo[col] = from_f32<T>(x[e] * inv - to_f32<T>(hi));
            }
        }
        if (tx == 0) a.lse[((int64_t)b * a.H + h) * a.Nq + i] = m[r] + logf(l[r]);
    }
}

// MODE 0: 32 keys stay, tiles of 64 queries that see any of them go by, head after head of the K/V head's; dK and dV.
// MODE 1: 32 queries stay, tiles of 64 keys of their hull go by; dQ.
template <typename T, int MODE, int DC>
__global__ void __launch_bounds__(NT) ruled_bwd_kernel(const RuledArgs a) {
    constexpr int P = DC + 4, N = DC / 32;
    extern __shared__ __align__(16) float smem[];
    float* X0 = smem;                          // K or Q
    float* X1 = X0 + BX * P;                   // V or dO
    float* Y = X1 + BX * P;                    // [2][Q, dO or K, V]
    float* Ps = Y + 4 * BY * P;
    float* Ds = Ps + BX * SLD;
    const int ty = group_of_four(), tx = column_of_group(), lane = threadIdx.x & 31;
    const int tile = MODE == 0 ? blockIdx.x : gridDim.x - 1 - blockIdx.x, b = blockIdx.z, group = a.H / a.Hkv, x0 = tile * BX;
    const int hk = MODE == 0 ? blockIdx.y : blockIdx.y / group, h_end = MODE == 0 ? (hk + 1) * group : blockIdx.y + 1;
    const T* k = (const T*)a.k.ptr + b * a.k.stride_b + hk * a.k.stride_h;
    const T* v = (const T*)a.v.ptr + b * a.v.stride_b + hk * a.v.stride_h;
    auto q_of = [&](int h) { return (const T*)a.q.ptr + b * a.q.stride_b + h * a.q.stride_h; };
    auto g_of = [&](int h) { return (const T*)a.d_o.ptr + b * a.d_o.stride_b + h * a.d_o.stride_h; };

    // the tiles that go by: [begin, end) of every head, those that matter found a lane a tile
    int h = MODE == 0 ? hk * group : blockIdx.y, begin, end;
    int2 hull = make_int2(0, 0);
    if (MODE == 0) {
        const int2 seen = a.rules.k_tiles[b * a.rules.k_tiles_b + x0 / 128];
        const int tiles = (a.Nq + BY - 1) / BY;
        begin = min(max(seen.x, 0), tiles) * (128 / BY);
        end = min(tiles, min(seen.y, tiles) * (128 / BY));
    } else {
        hull = hull_of<BX>(a, b, tile);
        begin = hull.x / BY;
        end = (hull.y + BY - 1) / BY;
    }
    int window = begin - 32, at = 0;
    uint32_t left = 0;
    auto next = [&] {                          // the next tile: of head h, number `at`; false: no more
        while (left == 0) {
            window += 32;
            if (window >= end) { ++h; window = begin; }
            if (h >= h_end || begin >= end) return false;
            bool there = window + lane < end;
            if (MODE == 0 && there) {
                const int2 sees = hull_of<BY>(a, b, window + lane);
                there = sees.x < x0 + BX && sees.y > x0;
            }
            left = __ballot_sync(0xffffffffu, there);
        }
        at = window + __ffs(left) - 1;
        left &= left - 1;
        return true;
    };
    auto copy_y = [&](int stage) {
        float* to = Y + stage * 2 * BY * P;
        if (MODE == 0) {
            copy_rows<T, DC, BY>(to, q_of(h), a.q.stride_n, at * BY, 0, a.Nq, a.D, a.pieces);
            copy_rows<T, DC, BY>(to + BY * P, g_of(h), a.d_o.stride_n, at * BY, 0, a.Nq, a.D, a.pieces);
        } else {
            copy_rows<T, DC, BY>(to, k, a.k.stride_n, at * BY, hull.x, hull.y, a.D, a.pieces);
            copy_rows<T, DC, BY>(to + BY * P, v, a.v.stride_n, at * BY, hull.x, hull.y, a.D, a.pieces);
        }
    };

    // what the four queries of a thread's rows (MODE 1) or columns (MODE 0) see, and their vectors
    RowRule rule[4];
    float lse[4], delta[4], slope = 0.f;
    auto queries = [&](int head, int i0, int step) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = i0 + step * e;
            const int64_t n = ((int64_t)b * a.H + head) * a.Nq + i;
            rule[e] = row_rule(a, b, i);
            lse[e] = i < a.Nq ? a.lse[n] : 0.f;
            delta[e] = i < a.Nq ? a.delta[n] : 0.f;
        }
        slope = a.rules.slopes ? a.rules.slopes[head] : 0.f;
    };
    if (MODE == 0) {
        copy_rows<T, DC, BX>(X0, k, a.k.stride_n, x0, 0, a.Nk, a.D, a.pieces);
        copy_rows<T, DC, BX>(X1, v, a.v.stride_n, x0, 0, a.Nk, a.D, a.pieces);
    } else {
        copy_rows<T, DC, BX>(X0, q_of(h), a.q.stride_n, x0, 0, a.Nq, a.D, a.pieces);
        copy_rows<T, DC, BX>(X1, g_of(h), a.d_o.stride_n, x0, 0, a.Nq, a.D, a.pieces);
        queries(h, x0 + ty * 4, 1);
    }
    uint64_t acc0[4][N], acc1[4][N];           // MODE 0: dK, dV; MODE 1: dQ
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int g = 0; g < N; ++g) { acc0[r][g] = 0; acc1[r][g] = 0; }

    bool there = next();
    if (there) copy_y(0);
    for (int stage = 0; there; stage ^= 1) {
        const float* Y0 = Y + stage * 2 * BY * P;
        const float* Y1 = Y0 + BY * P;
        const int y0 = at * BY;
        if (MODE == 0) queries(h, y0 + tx, 16);
        cp_async_wait();
        __syncthreads();                       // the tile is there, the other stage given back
        there = next();
        if (there) copy_y(stage ^ 1);
        uint64_t s2[4][4] = {}, p2[4][4] = {};
        dots<DC>(s2, X0, Y0, ty, tx);
        dots<DC>(p2, X1, Y1, ty, tx);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int e = MODE == 0 ? c : r, j = MODE == 0 ? x0 + ty * 4 + r : y0 + tx + 16 * c;
                float p = 0.f, ds = 0.f;
                if (j >= rule[e].first && j < rule[e].end) {
                    float dx;
                    const float x = ruled_score(a.rules.cap, slope, f2_sum(s2[r][c]) * a.scale, rule[e].position, j, dx);
                    p = expf(x - lse[e]);
                    ds = p * (f2_sum(p2[r][c]) - delta[e]) * dx;
                }
                const int at_s = (ty * 4 + r) * SLD + tx + 16 * c;
                if (MODE == 0) Ps[at_s] = p;
                Ds[at_s] = ds;
            }
        __syncwarp();                          // (a half-warp's own rows)
        weigh<DC>(acc0, Ds, Y0, ty, tx);
        if (MODE == 0) weigh<DC>(acc1, Ps, Y1, ty, tx);
        __syncwarp();
    }
    cp_async_wait();

#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int row = x0 + ty * 4 + r;
        if (row >= (MODE == 0 ? a.Nk : a.Nq)) continue;
        const fa_b200_tensor& t = MODE == 0 ? a.dk : a.dq;
        T* out0 = (T*)t.ptr + b * t.stride_b + row * t.stride_n + (MODE == 0 ? hk : (int)blockIdx.y) * t.stride_h;
        T* out1 = MODE == 0 ? (T*)a.dv.ptr + b * a.dv.stride_b + row * a.dv.stride_n + hk * a.dv.stride_h : nullptr;
#pragma unroll
        for (int g = 0; g < N; ++g) {
            float x[2], z[2];
            f2_unpack(acc0[r][g], x[0], x[1]);
            f2_unpack(acc1[r][g], z[0], z[1]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int col = column_of<DC>(tx, g) + e;
                if (col >= a.D) continue;
                out0[col] = from_f32<T>(x[e] * a.scale);
                if (MODE == 0) out1[col] = from_f32<T>(z[e]);
            }
        }
    }
}

RuledArgs make_args(const fa_b200_params& p, const float* delta, const Rules& rules) {
    RuledArgs a;
    a.q = p.q; a.k = p.k; a.v = p.v; a.o = p.o; a.o_lo = p.o_lo; a.d_o = p.d_o; a.dq = p.dq; a.dk = p.dk; a.dv = p.dv;
    a.lse = p.lse; a.delta = delta;
    a.B = p.B; a.Nq = p.Nq; a.Nk = p.Nk; a.H = p.H; a.Hkv = p.Hkv; a.D = p.D;
    a.scale = p.scale;
    a.rules = rules;
    bool pieces = p.dtype == FA_B200_F32 && p.D % 4 == 0;
    for (const fa_b200_tensor& t : {p.q, p.k, p.v, p.d_o})
        pieces = pieces && ((uintptr_t)t.ptr & 15u) == 0 && (t.stride_b | t.stride_n | t.stride_h) % 4 == 0;
    a.pieces = pieces;
    return a;
}

template <typename K>
int launch(K kernel, dim3 grid, size_t smem, const RuledArgs& a, void* stream) {
    FA_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    kernel<<<grid, NT, smem, (cudaStream_t)stream>>>(a);
    FA_CUDA_CHECK(cudaGetLastError());
    return FA_OK;
}

template <typename T, int DC>
int fwd(const fa_b200_params& p, const Rules& rules) {
    constexpr size_t smem = ((BX + 2 * BY) * (DC + 4) + BX * SLD) * sizeof(float);
    return launch(ruled_fwd_kernel<T, DC>, dim3((p.Nq + BX - 1) / BX, p.H, p.B), smem, make_args(p, nullptr, rules), p.stream);
}
template <typename T, int DC>
int bwd(const fa_b200_params& p, const float* delta, const Rules& rules) {
    constexpr size_t smem = ((2 * BX + 4 * BY) * (DC + 4) + 2 * BX * SLD) * sizeof(float);
    static_assert(smem <= 232448, "shared-memory plan does not fit");
    const RuledArgs a = make_args(p, delta, rules);
    const int phases = p.bwd_phases ? p.bwd_phases : 7;
    int rc = FA_OK;
    if (phases & 2) rc = launch(ruled_bwd_kernel<T, 0, DC>, dim3((p.Nk + BX - 1) / BX, p.Hkv, p.B), smem, a, p.stream);
    if (!rc && (phases & 4)) rc = launch(ruled_bwd_kernel<T, 1, DC>, dim3((p.Nq + BX - 1) / BX, p.H, p.B), smem, a, p.stream);
    return rc;
}
template <typename T>
int fwd_by_size(const fa_b200_params& p, const Rules& rules) {
    return p.D <= 32 ? fwd<T, 32>(p, rules) : (p.D <= 64 ? fwd<T, 64>(p, rules) : fwd<T, 128>(p, rules));
}
template <typename T>
int bwd_by_size(const fa_b200_params& p, const float* delta, const Rules& rules) {
    return p.D <= 32 ? bwd<T, 32>(p, delta, rules) : (p.D <= 64 ? bwd<T, 64>(p, delta, rules) : bwd<T, 128>(p, delta, rules));
}

}  // namespace

int simt_rules_fwd(const fa_b200_params& p, const Rules& rules) {
    switch (p.dtype) {
        case FA_B200_F16:  return fwd_by_size<__half>(p, rules);
        case FA_B200_BF16: return fwd_by_size<__nv_bfloat16>(p, rules);
        case FA_B200_F32:  return fwd_by_size<float>(p, rules);
    }
    return FA_EINVAL;
}

int simt_rules_bwd(const fa_b200_params& p, const float* delta, const Rules& rules) {
    switch (p.dtype) {
        case FA_B200_F16:  return bwd_by_size<__half>(p, delta, rules);
        case FA_B200_BF16: return bwd_by_size<__nv_bfloat16>(p, delta, rules);
        case FA_B200_F32:  return bwd_by_size<float>(p, delta, rules);
    }
    return FA_EINVAL;
}

}  // namespace fa
