// Rotary positions: pairs of columns of every head turned by position * frequency (the definition is in fa_b200.h).
//
// A block takes kTokens tokens.  Its threads first put the tokens' cosines and sines into shared memory, a pair's once for
// all heads of q and k: the angle and its reduction by whole turns in 64 bits (at position 10^6 a float angle would be
// off by 0.06), sine and cosine of what is left in 32.  Then a thread's unit is one 16-byte piece of a head (two of them,
// u and w, where the halves of the head are paired), read, turned and written.  Everything is read once and written once:
// memory bounds it, and for a token or two the launch.
#include "fa_common.cuh"
#include <type_traits>

namespace fa {
namespace {

struct RotaryArgs {
    fa_b200_tensor x[2], y[2];
    int heads[2];
    const void* positions;
    int64_t pos_sb, pos_sn, position0;
    const double* inv_freq;
    int pos64, N, D, half, interleaved;
    int64_t tokens;                // B * N
    float factor, sign;
};

constexpr int kThreads = 256;
constexpr int kMaxHalf = 64;       // head sizes up to 128

template <typename T, int VEC> struct Piece { T v[VEC]; };
template <typename T, int VEC>
__device__ __forceinline__ Piece<T, VEC> load_piece(const T* p) {
    Piece<T, VEC> r;
    if constexpr (VEC == 1) r.v[0] = *p;
    else *reinterpret_cast<uint4*>(&r) = *reinterpret_cast<const uint4*>(p);
    return r;
}
template <typename T, int VEC>
__device__ __forceinline__ void store_piece(T* p, const Piece<T, VEC>& r) {
    if constexpr (VEC == 1) *p = r.v[0];
    else *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&r);
}

// VEC elements a piece: 16 bytes, or one where addresses, head size or the number of pairs do not allow pieces.
template <typename T, int VEC, bool INTERLEAVED, int TOKENS>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryArgs a) {
    __shared__ float2 turn[TOKENS][kMaxHalf];            // factor * cos, factor * sin
    const int64_t token0 = (int64_t)blockIdx.x * TOKENS;
    const int n_tokens = (int)(a.tokens - token0 < TOKENS ? a.tokens - token0 : TOKENS);
    for (int e = threadIdx.x; e < n_tokens * a.half; e += kThreads) {
        const int t = e / a.half, i = e - t * a.half;
        const int64_t token = token0 + t, b = token / a.N, n = token - b * a.N;
        int64_t pos = a.position0 + n;
        if (a.positions) {
            const int64_t at = b * a.pos_sb + n * a.pos_sn;
            pos = a.pos64 ? ((const int64_t*)a.positions)[at] : ((const int32_t*)a.positions)[at];
        }
        const double angle = (double)pos * a.inv_freq[i];
        // less whole turns: 2 pi as a double and the rest of it
        const double turns = rint(angle * 0.15915494309189533577);
        const double rest = fma(-turns, 2.4492935982947064e-16, fma(-turns, 6.2831853071795864769, angle));
        float s, c;
        sincosf((float)rest, &s, &c);
        turn[t][i] = make_float2(a.factor * c, a.factor * a.sign * s);
    }
    __syncthreads();
    // units of a head: the pairs' pieces, then the copied ones
    const int n_turned = INTERLEAVED && VEC > 1 ? 2 * a.half / VEC : a.half / (VEC > 1 ? VEC : 1);
    const int in_place = a.x[0].ptr == a.y[0].ptr && (a.x[1].ptr == a.y[1].ptr);
    const int n_units = n_turned + (in_place ? 0 : (a.D - 2 * a.half) / VEC);
    const int heads = a.heads[0] + a.heads[1];
    const int total = n_tokens * heads * n_units;
#pragma unroll 4
    for (int e = threadIdx.x; e < total; e += kThreads) {
        const int row = e / n_units, unit = e - row * n_units;
        const int t = row / heads, hh = row - t * heads;
        const int which = hh >= a.heads[0];
        const int h = which ? hh - a.heads[0] : hh;
        const int64_t token = token0 + t, b = token / a.N, n = token - b * a.N;
        const fa_b200_tensor& xt = a.x[which];
        const fa_b200_tensor& yt = a.y[which];
        const T* x = (const T*)xt.ptr + b * xt.stride_b + n * xt.stride_n + h * xt.stride_h;
        T* y = (T*)yt.ptr + b * yt.stride_b + n * yt.stride_n + h * yt.stride_h;
        if (unit >= n_turned) {
            const int c = 2 * a.half + (unit - n_turned) * VEC;
            store_piece<T, VEC>(y + c, load_piece<T, VEC>(x + c));
        } else if (INTERLEAVED && VEC > 1) {
            const int c = unit * VEC;
            Piece<T, VEC> p = load_piece<T, VEC>(x + c);
#pragma unroll
            for (int v = 0; v < VEC; v += 2) {
                const float2 cs = turn[t][c / 2 + v / 2];
                const float u = to_f32<T>(p.v[v]), w = to_f32<T>(p.v[v + 1]);
                p.v[v] = from_f32<T>(u * cs.x - w * cs.y);
                p.v[v + 1] = from_f32<T>(w * cs.x + u * cs.y);
            }
            store_piece<T, VEC>(y + c, p);
        } else {
            const int i = unit * VEC;
            const int c0 = INTERLEAVED ? 2 * i : i, c1 = INTERLEAVED ? 2 * i + 1 : i + a.half;
            Piece<T, VEC> pu = load_piece<T, VEC>(x + c0), pw = load_piece<T, VEC>(x + c1);
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const float2 cs = turn[t][i + v];
                const float u = to_f32<T>(pu.v[v]), w = to_f32<T>(pw.v[v]);
                pu.v[v] = from_f32<T>(u * cs.x - w * cs.y);
                pw.v[v] = from_f32<T>(w * cs.x + u * cs.y);
            }
            store_piece<T, VEC>(y + c0, pu);
            store_piece<T, VEC>(y + c1, pw);
        }
    }
}

template <typename T, int VEC, bool INTERLEAVED>
int launch(const RotaryArgs& a, cudaStream_t st) {
    constexpr int kTokens = 4;
    const int64_t blocks = (a.tokens + kTokens - 1) / kTokens;
    if (blocks > 0x7fffffff) { set_error("rotary: too many tokens"); return FA_EUNSUPPORTED; }
    rotary_kernel<T, VEC, INTERLEAVED, kTokens><<<(unsigned)blocks, kThreads, 0, st>>>(a);
    FA_CUDA_CHECK(cudaGetLastError());
    return FA_OK;
}

template <typename T>
int pick(const RotaryArgs& a, bool pieces, cudaStream_t st) {
    constexpr int V = 16 / (int)sizeof(T);
    if (pieces) return a.interleaved ? launch<T, V, true>(a, st) : launch<T, V, false>(a, st);
    return a.interleaved ? launch<T, 1, true>(a, st) : launch<T, 1, false>(a, st);
}

}  // namespace
}  // namespace fa

using namespace fa;

extern "C" int fa_b200_rotary(const fa_b200_rotary_params* p) {
    if (!p) { set_error("params is null"); return FA_EINVAL; }
    if (p->struct_bytes != sizeof(fa_b200_rotary_params)) {
        set_error("struct_bytes %zu does not match this library's fa_b200_rotary_params (%zu bytes)", p->struct_bytes, sizeof(fa_b200_rotary_params));
        return FA_EINVAL;
    }
    const bool two = p->x[1].ptr != nullptr;
    if (p->B < 0 || p->N < 0 || p->heads[0] < 0 || (two && p->heads[1] < 0) || p->D <= 0) { set_error("rotary: negative size"); return FA_EINVAL; }
    if (p->D > 2 * kMaxHalf) { set_error("rotary: head_dim %d is not supported (maximum %d)", p->D, 2 * kMaxHalf); return FA_EUNSUPPORTED; }
    if (p->half < 0 || 2 * p->half > p->D) { set_error("rotary: %d pairs do not fit a head of %d", p->half, p->D); return FA_EINVAL; }
    if (p->dtype != FA_B200_F16 && p->dtype != FA_B200_BF16 && p->dtype != FA_B200_F32) { set_error("unknown dtype %d", p->dtype); return FA_EINVAL; }
    if (!(p->factor == p->factor)) { set_error("rotary: factor is NaN"); return FA_EINVAL; }
    if (p->B == 0 || p->N == 0 || p->heads[0] + (two ? p->heads[1] : 0) == 0) return FA_OK;
    if ((p->heads[0] > 0 && (!p->x[0].ptr || !p->y[0].ptr)) || (two && !p->y[1].ptr)) { set_error("rotary: null pointer"); return FA_EINVAL; }
    if (p->half > 0 && !p->inv_freq) { set_error("rotary: inv_freq is null"); return FA_EINVAL; }
    RotaryArgs a;
    const int eb = (int)dtype_bytes(p->dtype), vec = 16 / eb;
    bool pieces = p->D % vec == 0 && (p->interleaved ? 2 * p->half : p->half) % vec == 0;
    for (int i = 0; i < 2; ++i) {
        a.x[i] = p->x[i]; a.y[i] = p->y[i];
        a.heads[i] = i == 0 || two ? p->heads[i] : 0;
        if (a.heads[i] == 0) continue;
        for (const fa_b200_tensor& t : {p->x[i], p->y[i]})
            if (((uintptr_t)t.ptr & 15u) != 0 || (a.heads[i] > 1 && t.stride_h % vec) || (p->N > 1 && t.stride_n % vec) || (p->B > 1 && t.stride_b % vec)) pieces = false;
    }
    if (!two) { a.x[1] = a.x[0]; a.y[1] = a.y[0]; }
    a.positions = p->positions; a.pos_sb = p->positions_stride_b; a.pos_sn = p->positions_stride_n; a.position0 = p->position0;
    a.pos64 = p->positions_64bit; a.inv_freq = p->inv_freq;
    a.N = p->N; a.D = p->D; a.half = p->half; a.interleaved = p->interleaved;
    a.tokens = (int64_t)p->B * p->N;
    a.factor = p->factor; a.sign = p->inverse ? -1.f : 1.f;
    GuardDevice g(p->device);
    if (!g.ok) { set_error("cudaSetDevice(%d) failed", p->device); return FA_ECUDA; }
    cudaStream_t st = (cudaStream_t)p->stream;
    if (p->dtype == FA_B200_F32) return pick<float>(a, pieces, st);
    return p->dtype == FA_B200_BF16 ? pick<__nv_bfloat16>(a, pieces, st) : pick<__half>(a, pieces, st);
}
