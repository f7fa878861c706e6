// Rotary positions: pairs of columns of every head turned by position * frequency (the definition is in fa_b200.h).
//
// A block takes a few tokens.  Its threads ask for their pieces of the heads first, and while those are on their way put the
// tokens' cosines and sines into shared memory, a pair's once for all heads of q and k: the angle and its reduction by whole
// turns in 64 bits (at position 10^6 a float angle would be off by 0.06), sine and cosine of the part of a turn that is left
// in 32.  A unit is one 16-byte piece of a head, or two of them, u and w, where the halves of the head are paired.  Everything
// is read once and written once: memory bounds it, and for a token or two the launch.  B4 N4096 H32 on 8 D128 bf16, there and back:
// 116 us, 0.90 of the rate of a copy; one token of each of 32 requests 8 us.
#include "fa_common.cuh"
#include "sm100_ptx.cuh"
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
constexpr int kAtOnce = 4;         // units a thread has on their way
constexpr int kPasses = 2;
constexpr int kMaxTurns = 1024;    // tokens times pairs of a block
constexpr int kMaxTokens = 64;     // ... and tokens

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Piece { T v[VEC]; };
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

// Elements at, at + 1 of a piece as floats, and back.
template <typename T, int VEC>
__device__ __forceinline__ void get2(const Piece<T, VEC>& p, int at, float& x, float& y) {
    if constexpr (sizeof(T) == 4) { x = to_f32<T>(p.v[at]); y = to_f32<T>(p.v[at + 1]); }
    else ptx::unpack2<std::is_same<T, __nv_bfloat16>::value>(reinterpret_cast<const uint32_t*>(&p)[at / 2], x, y);
}
template <typename T, int VEC>
__device__ __forceinline__ void put2(Piece<T, VEC>& p, int at, float x, float y) {
    if constexpr (sizeof(T) == 4) { p.v[at] = from_f32<T>(x); p.v[at + 1] = from_f32<T>(y); }
    else reinterpret_cast<uint32_t*>(&p)[at / 2] = ptx::pack2<std::is_same<T, __nv_bfloat16>::value>(x, y);
}

// VEC elements a piece: 16 bytes, or one where addresses, head size or the number of pairs do not allow pieces.
template <typename T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryArgs a, int tokens_per_block) {
    // factor * cos and factor * sin of a token's pairs.  A unit's pairs v, v + 1 side by side, the units of one v next to each
    // other: a warp's 8-byte loads go to different banks (in the pairs' order every load took four turns).
    __shared__ __align__(8) float cos_of[kMaxTurns], sin_of[kMaxTurns];
    __shared__ int64_t base_of[kMaxTokens][4];           // a token's place in x[0], x[1], y[0], y[1]
    __shared__ int2 place[kMaxTokens];                   // its batch entry and row
    const int64_t token0 = (int64_t)blockIdx.x * tokens_per_block;
    const int n_tokens = (int)(a.tokens - token0 < tokens_per_block ? a.tokens - token0 : tokens_per_block);
    // units of a head: the pairs' pieces, then the copied ones
    constexpr bool ONE = INTERLEAVED && VEC > 1;         // a unit is one piece
    const int n_turned = ONE ? 2 * a.half / VEC : a.half / VEC;
    const bool in_place = a.x[0].ptr == a.y[0].ptr && a.x[1].ptr == a.y[1].ptr;
    const int n_units = n_turned + (in_place ? 0 : (a.D - 2 * a.half) / VEC);
    const int heads = a.heads[0] + a.heads[1];
    const int n_units_or_1 = n_units > 0 ? n_units : 1;

    // A thread keeps its unit and goes through the rows (token, head), `step` rows at a time: no division behind the first ones
    // (with them, 64-bit ones among them, the kernel took 150 us where it takes 60).
    const int step = kThreads / n_units_or_1, unit = (int)threadIdx.x % n_units_or_1;
    const int rows = n_tokens * heads, first = (int)threadIdx.x / n_units_or_1;
    const bool idle = n_units == 0 || first >= step;     // (threads beyond whole rows)
    if (threadIdx.x < (unsigned)n_tokens) {
        const uint32_t token = (uint32_t)token0 + threadIdx.x, b = token / (uint32_t)a.N, n = token - b * (uint32_t)a.N;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            base_of[threadIdx.x][w] = (int64_t)b * a.x[w].stride_b + (int64_t)n * a.x[w].stride_n;
            base_of[threadIdx.x][2 + w] = (int64_t)b * a.y[w].stride_b + (int64_t)n * a.y[w].stride_n;
        }
        place[threadIdx.x] = make_int2((int)b, (int)n);
    }
    __syncthreads();
    int t = 0, hh = first;
    while (hh >= heads) { hh -= heads; ++t; }
    // columns of a unit's first and second piece (the second: halves, or single columns of interleaved pairs)
    auto col0 = [&](int unit) { return unit >= n_turned ? 2 * a.half + (unit - n_turned) * VEC : (INTERLEAVED && VEC == 1 ? 2 * unit : unit * VEC); };
    auto col1 = [&](int unit) { return INTERLEAVED ? 2 * unit + 1 : unit * VEC + a.half; };

    const bool turned = unit < n_turned;
    const int c0 = col0(unit), c1 = col1(unit);
    constexpr int P = VEC == 1 ? 1 : (ONE ? VEC / 2 : VEC);          // pairs of a unit
    auto slot = [&](int i) { return P == 1 ? i : ((i % P / 2) * n_turned + i / P) * 2 + (i & 1); };
    for (int row0 = first, pass = 0; pass == 0 || row0 - first < rows; row0 += step * kAtOnce, ++pass) {
        Piece<T, VEC> pu[kAtOnce], pw[kAtOnce];
        T* y[kAtOnce];
        int tt[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            if (idle || row0 + k * step >= rows) continue;
            const int which = hh >= a.heads[0], h = which ? hh - a.heads[0] : hh;
            const T* x = (const T*)a.x[which].ptr + base_of[t][which] + h * a.x[which].stride_h;
            y[k] = (T*)a.y[which].ptr + base_of[t][2 + which] + h * a.y[which].stride_h;
            tt[k] = t;
            pu[k] = load_piece<T, VEC>(x + c0);
            if (!ONE && turned) pw[k] = load_piece<T, VEC>(x + c1);
            hh += step;
            while (hh >= heads) { hh -= heads; ++t; }
        }
        if (pass == 0) {
            for (int e = threadIdx.x; e < n_tokens * a.half; e += kThreads) {
                const int at = e / a.half, i = e - at * a.half;
                const int2 bn = place[at];
                int64_t pos = a.position0 + bn.y;
                if (a.positions) {
                    const int64_t from = bn.x * a.pos_sb + bn.y * a.pos_sn;
                    pos = a.pos64 ? ((const int64_t*)a.positions)[from] : ((const int32_t*)a.positions)[from];
                }
                const double turns = (double)pos * a.inv_freq[i] * 0.15915494309189533577;       // 1 / 2 pi
                float s, c;
                sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
                cos_of[at * a.half + slot(i)] = a.factor * c;
                sin_of[at * a.half + slot(i)] = a.factor * a.sign * s;
            }
            __syncthreads();
        }
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            if (idle || row0 + k * step >= rows) continue;
            if (turned) {
                const float *cs = cos_of + tt[k] * a.half, *sn = sin_of + tt[k] * a.half;
                if constexpr (VEC == 1) {
                    const float x = to_f32<T>(pu[k].v[0]), w = to_f32<T>(pw[k].v[0]), c = cs[unit], n = sn[unit];
                    pu[k].v[0] = from_f32<T>(x * c - w * n);
                    pw[k].v[0] = from_f32<T>(w * c + x * n);
                } else {
#pragma unroll
                    for (int v = 0; v < P; v += 2) {
                        // two pairs at once: u and w of both
                        const uint64_t c2 = *reinterpret_cast<const uint64_t*>(cs + ((v / 2) * n_turned + unit) * 2);
                        const uint64_t s2 = *reinterpret_cast<const uint64_t*>(sn + ((v / 2) * n_turned + unit) * 2);
                        float u0, u1, w0, w1;
                        if constexpr (ONE) { get2(pu[k], 2 * v, u0, w0); get2(pu[k], 2 * v + 2, u1, w1); }
                        else { get2(pu[k], v, u0, u1); get2(pw[k], v, w0, w1); }
                        const uint64_t u = ptx::f2_pack(u0, u1), w = ptx::f2_pack(w0, w1);
                        ptx::f2_unpack(ptx::f2_fma(w, s2 ^ 0x8000000080000000ull, ptx::f2_mul(u, c2)), u0, u1);
                        ptx::f2_unpack(ptx::f2_fma(u, s2, ptx::f2_mul(w, c2)), w0, w1);
                        if constexpr (ONE) { put2(pu[k], 2 * v, u0, w0); put2(pu[k], 2 * v + 2, u1, w1); }
                        else { put2(pu[k], v, u0, u1); put2(pw[k], v, w0, w1); }
                    }
                }
                if (!ONE) store_piece<T, VEC>(y[k] + c1, pw[k]);
            }
            store_piece<T, VEC>(y[k] + c0, pu[k]);
        }
    }
}

template <typename T, int VEC, bool INTERLEAVED>
int launch(const RotaryArgs& a, int device, cudaStream_t st) {
    // tokens for a few passes of what a block's threads have on their way, fewer where that would leave SMs idle
    const int64_t heads = a.heads[0] + a.heads[1];
    const int64_t units = heads * ((INTERLEAVED && VEC > 1 ? 2 * a.half / VEC : a.half / VEC) + (a.D - 2 * a.half) / VEC);
    int64_t tokens = units > 0 ? (int64_t)kThreads * kAtOnce * kPasses / units : 1;
    const int64_t spread = a.tokens / (4 * (int64_t)(sm_count(device) > 0 ? sm_count(device) : 1));
    if (tokens > spread) tokens = spread;
    if (a.half > 0 && tokens > kMaxTurns / a.half) tokens = kMaxTurns / a.half;
    if (tokens > kMaxTokens) tokens = kMaxTokens;
    if (tokens < 1) tokens = 1;
    const int64_t blocks = (a.tokens + tokens - 1) / tokens;
    if (a.tokens > 0x7fffffff || heads * a.D * tokens > 0x3fffffff) { set_error("rotary: too many tokens or heads"); return FA_EUNSUPPORTED; }
    rotary_kernel<T, VEC, INTERLEAVED><<<(unsigned)blocks, kThreads, 0, st>>>(a, (int)tokens);
    FA_CUDA_CHECK(cudaGetLastError());
    return FA_OK;
}

template <typename T>
int pick(const RotaryArgs& a, bool pieces, int device, cudaStream_t st) {
    constexpr int V = 16 / (int)sizeof(T);
    if (pieces) return a.interleaved ? launch<T, V, true>(a, device, st) : launch<T, V, false>(a, device, st);
    return a.interleaved ? launch<T, 1, true>(a, device, st) : launch<T, 1, false>(a, device, st);
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
    if (p->dtype == FA_B200_F32) return pick<float>(a, pieces, p->device, st);
    return p->dtype == FA_B200_BF16 ? pick<__nv_bfloat16>(a, pieces, p->device, st) : pick<__half>(a, pieces, p->device, st);
}
