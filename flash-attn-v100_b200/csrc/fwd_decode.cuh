// Attention under rules for one new token a request, or a few: up to 16 rows (queries times the heads of a K/V head) against
// a long cache.  Part of fwd_sm100.cu's RULES instances, with its split schedule: one range of (pair, key block) units a CTA.
//
// What bounds it is reading K and V once; a tcgen05 tile would have 128 rows, of which a decoding call uses 1 to 16, all in one
// warp's lanes of tensor memory, and that warp's 128 exponentials a row would be the step (32 requests of 2048-8192 keys,
// H32 Hkv8 D128 bf16, cap and distances: 207 us, here 124 to 139 from one GPU to another, 106 at the copy rate).  So the
// small matrix instruction instead: each of eight warps takes 16 keys of a 128-key block, S (16 x 16) = Q K^T with Q in
// registers and K by ldmatrix from the tile TMA has brought, its own running maximum and sum, O (16 x D) += P V in registers.
// A warp never waits for another one until a stretch ends, when the eight are put together through shared memory.  P is
// a pair of values of the call's type, hi + lo (two products), so that its rounding stays below the output's (as one value an
// fp16 call was off by 2.9e-4 of its outputs where their own rounding is 2.1e-4; 32 requests 144 -> 147 us).
// Sixteen warps (registers then spill: 202 us), 8-row registers (no change) and, at D 64, two blocks a warp at once (no
// change) brought nothing; D 64 gets 62 % of D 128's rate out of a cache whose heads lie side by side, 128 bytes a head.
#pragma once

template <int D>
struct DecodeCfg {
    static constexpr int kNBox = D / 64, kTileBytes = kNBox * kBoxBytes;
    static constexpr int kStages = D == 128 ? 3 : 6;               // blocks of K and V on their way: 192 KB
    static constexpr int kWarps = 8;
    static constexpr int kFull = 0;                                // [2][kStages]: K, V
    static constexpr int kEmpty = 2 * kStages;                     // [kStages], one arrival per warp
    static constexpr int kNumBars = 3 * kStages;
    static constexpr int kSumBytes = kWarps * 8 * D * 4;           // eight rows of every warp's O
    static constexpr int kMlBytes = kWarps * 16 * 8;               // maximum and sum of 16 rows
    static constexpr int kSmemBytes = 2 * kStages * kTileBytes + kSumBytes + kMlBytes + kNumBars * 8 + 64 + 1024;
    static_assert(kSmemBytes <= 232448, "shared-memory plan does not fit");
};

__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int D, bool BF16, int RULES>
__global__ void __launch_bounds__(288, 1)
fwd_decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const FwdArgs a) {
    using Cfg = DecodeCfg<D>;
    using T16 = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
    constexpr int ST = Cfg::kStages, TILE = Cfg::kTileBytes, KS = D / 16;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* sK = smem;
    uint8_t* sV = sK + ST * TILE;
    float* sO = (float*)(sV + ST * TILE);                          // [warp][8 rows][D]
    float2* sMl = (float2*)((uint8_t*)sO + Cfg::kSumBytes);        // [warp][16 rows]
    uint64_t* bars = (uint64_t*)((uint8_t*)sMl + Cfg::kMlBytes);
    volatile uint32_t* abort_flag = (volatile uint32_t*)(bars + Cfg::kNumBars);
    volatile RangeStart* range = (volatile RangeStart*)(abort_flag + 4);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (warp == Cfg::kWarps) {
        if (lane < Cfg::kNumBars) mbar_init(&bars[lane], lane >= Cfg::kEmpty ? (uint32_t)Cfg::kWarps : 1u);
        if (lane == 0) {
            wait_control_init(abort_flag, a.wait_limit_ms);
            prefetch_tensormap(&map_k);
            prefetch_tensormap(&map_v);
        }
        fence_mbar_init();
    }
    if (warp == 0) find_range<2, RULES>(a, lane, range);
    __syncthreads();
    grid_launch_dependents();       // fwd_merge_kernel, which waits for this grid's end

    if (warp == Cfg::kWarps) {
        if (elect_one()) {
            int c = 0;
            bool ok = true;
            for (WorkLoop<2, RULES> wl(a, range); wl.more(a) && ok; wl.advance()) {
                Stretch st;
                wl.get(a, 0, st);
                const int hk = st.h * a.pack / (a.H / a.Hkv);
                for (int j = st.j0; j < st.j1 && ok; ++j, ++c) {
                    const int s = c % ST;
                    ok = mbar_wait(&bars[Cfg::kEmpty + s], ((uint32_t)(c / ST) & 1u) ^ 1u, abort_flag);
                    if (!ok) break;
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        mbar_expect_tx(&bars[Cfg::kFull + y * ST + s], TILE);
#pragma unroll
                        for (int bx = 0; bx < Cfg::kNBox; ++bx)
                            tma_load_4d((y ? sV : sK) + s * TILE + bx * kBoxBytes, y ? &map_v : &map_k, &bars[Cfg::kFull + y * ST + s], bx * 64, hk,
                                        j * kBlockN, st.b);
                    }
                }
            }
            // unwinding: copies in flight land before shared memory is given up
            for (int s = 0; s < ST && !ok; ++s) {
                const int n = (c + ST - 1 - s) / ST;
                for (int y = 0; y < 2; ++y)
                    for (int spin = 0; spin < 4096 && n > 0 && !mbar_try_wait(&bars[Cfg::kFull + y * ST + s], (uint32_t)(n - 1) & 1u); ++spin) {}
            }
        }
        __syncwarp();
    } else {
        auto meet = [] { asm volatile("barrier.cta.sync 1, 256;" ::: "memory"); };
        const int rows = a.pack * a.Nq;                            // at most 16
        const bool second = rows > 8;                              // rows 8-15 are there
        const int r0 = lane >> 2, l2 = (lane & 3) * 2;
        const uint32_t sK_u = smem_u32(sK), sV_u = smem_u32(sV);
        // my row of the 8 x 8 matrices ldmatrix loads: K: keys (0-7, 0-7, 8-15, 8-15), pieces (0, 1, 0, 1); V: keys (0-7, 8-15, ..)
        const int mi = lane >> 3, key_k = warp * 16 + (mi >> 1) * 8 + (lane & 7), key_v = warp * 16 + (mi & 1) * 8 + (lane & 7);
        auto piece = [](uint32_t tile, int key, int chunk) {       // 16-byte piece of a row: boxes of eight, swizzled by the row
            return tile + (uint32_t)(chunk >> 3) * kBoxBytes + (uint32_t)key * 128u + (uint32_t)(((chunk ^ key) & 7) << 4);
        };
        int c = 0;
        bool ok = true;                                            // (a wait that ran out: the walk goes on without waiting, to every meeting)
        if (threadIdx.x == 0) a.part_meta[blockIdx.x] = make_int4(0, 0, 0, 0);
        for (WorkLoop<2, RULES> wl(a, range); wl.more(a); wl.advance()) {
            Stretch st;
            wl.get(a, 0, st);
            const int64_t slot = 2 * (int64_t)blockIdx.x + (st.j0 == st.jb ? 1 : 0);
            if (threadIdx.x == 0 && !st.whole() && st.j0 == st.jb) {
                // the pair starts here and goes on in the ranges of the CTAs behind this one
                const int total = range->total, ctas = range->ctas;
                const int end = range_begin((int)blockIdx.x + 1, ctas, total) + (st.n[0] - st.j1);
                int k = 1;
                while (range_begin((int)blockIdx.x + k, ctas, total) < end) ++k;
                a.part_meta[blockIdx.x] = make_int4(st.b, st.h, st.pair, k);
            }
            const int2 seen = tile_hull(a, st.b, a.q_per_tile, 0, 0);
            int2 keys[2];
            int at[2];
            float slope[2];
            uint32_t qa[KS][4];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const int r = r0 + 8 * y, i = r / a.pack, h = st.h * a.pack + r % a.pack;
                const bool mine = r < rows;
                keys[y] = mine ? a.rules.rows[st.b * a.rules.rows_b + i] : make_int2(0, 0);
                at[y] = i + a.rules.origin[st.b * a.rules.origin_b];
                slope[y] = mine && a.rules.slopes ? a.rules.slopes[h] * kLog2e : 0.f;
                const T16* q = reinterpret_cast<const T16*>(a.q) + st.b * a.q_sb + i * a.q_sn + h * a.q_sh + l2;
#pragma unroll
                for (int kk = 0; kk < KS; ++kk)
#pragma unroll
                    for (int z = 0; z < 2; ++z)
                        qa[kk][y + 2 * z] = mine && kk * 16 + z * 8 < a.d ? *reinterpret_cast<const uint32_t*>(q + kk * 16 + z * 8) : 0u;
            }
            float acc[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;

            for (int j = st.j0; j < st.j1; ++j, ++c) {
                const int s = c % ST, key0 = j * kBlockN + warp * 16;
                const uint32_t ph = (uint32_t)(c / ST) & 1u;
                ok = ok && mbar_wait(&bars[Cfg::kFull + s], ph, abort_flag);
                ok = __all_sync(0xffffffffu, ok);
                const bool work = ok && key0 < seen.y && key0 + 16 > seen.x;        // some row may see one of my keys
                uint32_t ph_[4], pl_[4];
                if (work) {
                    float sc[2][4] = {};
#pragma unroll
                    for (int kk = 0; kk < KS; ++kk) {
                        if (kk * 16 >= a.d) break;
                        uint32_t b[4];
                        ldmatrix_x4(piece(sK_u + s * TILE, key_k, kk * 2 + (mi & 1)), b);
                        mma_16816<BF16>(sc[0], qa[kk], b[0], b[1]);
                        mma_16816<BF16>(sc[1], qa[kk], b[2], b[3]);
                    }
                    // x in log2 units, as the instances above have it
                    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int y = e >> 1, key = key0 + n * 8 + l2 + (e & 1);
                            if (y == 1 && !second) { sc[n][e] = -INFINITY; continue; }
                            float x = RULES == 2 ? tanh_any(sc[n][e] * a.cap_in) * a.cap_out : sc[n][e] * a.scale_log2;
                            x = fmaf(-slope[y], fabsf((float)(at[y] - key)), x);
                            if (key < keys[y].x || key >= keys[y].y) x = -INFINITY;
                            sc[n][e] = x;
                            top[y] = fmaxf(top[y], x);
                        }
                    bool grow = false;
                    float m_new[2];
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        top[y] = fmaxf(top[y], __shfl_xor_sync(0xffffffffu, top[y], 1));
                        top[y] = fmaxf(top[y], __shfl_xor_sync(0xffffffffu, top[y], 2));
                        m_new[y] = fmaxf(m[y], top[y]);
                        grow |= m_new[y] - m[y] > kRescaleThreshold;
                    }
                    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            const float alpha = m_new[y] == -INFINITY ? 0.f : ex2(m[y] - m_new[y]);
                            m[y] = m_new[y];
                            l[y] *= alpha;
#pragma unroll
                            for (int n = 0; n < D / 8; ++n) { acc[n][2 * y] *= alpha; acc[n][2 * y + 1] *= alpha; }
                        }
                    }
                    const float off[2] = {kPShift - (m[0] == -INFINITY ? 0.f : m[0]), kPShift - (m[1] == -INFINITY ? 0.f : m[1])};
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            const float p0 = ex2(sc[n][2 * y] + off[y]), p1 = ex2(sc[n][2 * y + 1] + off[y]);
                            l[y] += p0 + p1;
                            pack2_pair<BF16>(p0, p1, ph_[2 * n + y], pl_[2 * n + y]);
                        }
                }
                ok = ok && mbar_wait(&bars[Cfg::kFull + ST + s], ph, abort_flag);
                ok = __all_sync(0xffffffffu, ok);
                if (work && ok) {
                    // keys nobody sees: 0 times unwritten memory is no zero
                    const bool edge = key0 < seen.x || key0 + 16 > seen.y;
                    uint32_t keep[2];
#pragma unroll
                    for (int z = 0; z < 2; ++z) {
                        const int key = key0 + z * 8 + l2;
                        keep[z] = (key >= seen.x && key < seen.y ? 0xFFFFu : 0u) | (key + 1 >= seen.x && key + 1 < seen.y ? 0xFFFF0000u : 0u);
                    }
#pragma unroll
                    for (int n = 0; n < D / 16; ++n) {
                        if (n * 16 >= a.d) break;
                        uint32_t b[4];
                        ldmatrix_x4_trans(piece(sV_u + s * TILE, key_v, n * 2 + (mi >> 1)), b);
                        if (edge) { b[0] &= keep[0]; b[1] &= keep[1]; b[2] &= keep[0]; b[3] &= keep[1]; }
                        mma_16816<BF16>(acc[2 * n], ph_, b[0], b[1]);
                        mma_16816<BF16>(acc[2 * n + 1], ph_, b[2], b[3]);
                        mma_16816<BF16>(acc[2 * n], pl_, b[0], b[1]);
                        mma_16816<BF16>(acc[2 * n + 1], pl_, b[2], b[3]);
                    }
                }
                mbar_arrive_warp(&bars[Cfg::kEmpty + s]);
            }

            // ---- the eight warps' sums: maxima first, then eight rows of O at a time
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                l[y] += __shfl_xor_sync(0xffffffffu, l[y], 1);
                l[y] += __shfl_xor_sync(0xffffffffu, l[y], 2);
                if ((lane & 3) == 0) sMl[warp * 16 + r0 + 8 * y] = make_float2(m[y], l[y]);
            }
            meet();
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                if (y == 1 && !second) break;
                float top = -INFINITY;
#pragma unroll
                for (int w = 0; w < Cfg::kWarps; ++w) top = fmaxf(top, sMl[w * 16 + r0 + 8 * y].x);
                const float by = m[y] == -INFINITY ? 0.f : ex2(m[y] - top);
                float* mine = sO + (warp * 8 + r0) * D;
#pragma unroll
                for (int n = 0; n < D / 8; ++n)
                    *reinterpret_cast<float2*>(mine + ((n * 8 + l2) ^ (r0 * 8 & (D - 1)))) = make_float2(acc[n][2 * y] * by, acc[n][2 * y + 1] * by);
                // A thread four columns of a row (at D 64 half of the threads).  What it reads of the maxima and sums it reads before
                // it meets the others: a warp that has nothing to add up here may be through the next stretch, and write its own
                // maxima there, before this stretch's last sums are formed.  (The sums of O are written behind the next stretch's
                // first meeting.)
                static_assert(8 * (D / 4) <= 32 * Cfg::kWarps, "a thread has one piece at most");
                const int e = threadIdx.x, row = e / (D / 4), col = (e % (D / 4)) * 4, r = row + 8 * y;
                const bool adds = e < 8 * (D / 4) && r < rows;
                float big = -INFINITY, sum = 0.f;
                if (adds) {
#pragma unroll
                    for (int w = 0; w < Cfg::kWarps; ++w) big = fmaxf(big, sMl[w * 16 + r].x);
#pragma unroll
                    for (int w = 0; w < Cfg::kWarps; ++w) {
                        const float2 ml = sMl[w * 16 + r];
                        sum = fmaf(ml.x == -INFINITY ? 0.f : ex2(ml.x - big), ml.y, sum);
                    }
                }
                meet();
                if (adds) {
                    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int w = 0; w < Cfg::kWarps; ++w) {
                        const float4 x = *reinterpret_cast<const float4*>(sO + (w * 8 + row) * D + (col ^ (row * 8 & (D - 1))));
                        o.x += x.x; o.y += x.y; o.z += x.z; o.w += x.w;
                    }
                    if (!st.whole()) {
                        a.part_o[(slot * a.part_rows + r) * (D / 4) + col / 4] = o;
                        if (col == 0) a.part_ml[slot * a.part_rows + r] = make_float2(big, sum);
                    } else {
                        const int i = r / a.pack, h = st.h * a.pack + r % a.pack;
                        const float inv = big == -INFINITY ? 0.f : 1.f / sum;
                        if (col < a.d)
                            *reinterpret_cast<uint2*>(reinterpret_cast<T16*>(a.o) + st.b * a.o_sb + i * a.o_sn + h * a.o_sh + col) =
                                make_uint2(pack2<BF16>(o.x * inv, o.y * inv), pack2<BF16>(o.z * inv, o.w * inv));
                        if (col == 0) a.lse[((int64_t)st.b * a.H + h) * a.Nq + i] = kLn2 * ((big - kPShift) + log2f(sum));
                    }
                }
                if (y == 0 && second) meet();                      // the rows' room is written anew
            }
        }
    }
    __syncthreads();
    if (threadIdx.x == 0 && *abort_flag) report_status(a.status, 1);
}

// Put together what ranges cut: block (c, r) takes row r of the pair that starts in CTA c's range and goes on in others.  A
// thread holds four columns and every U-th part, so that a few parts are under way at once; the U sums are added in
// their order, which does not depend on which CTA finished first.  What bounds it is the latency of its loads (a lane a row, all
// parts one after another, as fwd_merge_kernel has it for tiles: 16 us for the 18 parts of one request's 4096 keys, H32 Hkv8 D128 bf16;
// the call 31 -> 18 us, with 16384 keys 43 -> 31).
template <int D, bool BF16>
__global__ void __launch_bounds__(128) fwd_decode_merge_kernel(const FwdArgs a) {
    using T16 = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
    constexpr int C = D / 4, U = 128 / C;
    __shared__ float4 sum_o[U][C];
    __shared__ float sum_l[U];
    const int c = blockIdx.x, r = blockIdx.y, u = threadIdx.x / C, col = threadIdx.x % C;
    auto at = [&](int k) { return (2 * ((int64_t)c + k) + (k == 0 ? 1 : 0)) * a.part_rows + r; };
    grid_dependency_wait();
    const int4 meta = a.part_meta[c];
    // (read before the record is there: a part that is none is not used)
    const int64_t first = at(c + u < (int)gridDim.x ? u : 0);
    const float2 ml0 = a.part_ml[first];
    const float4 o0 = a.part_o[first * C + col];
    if (meta.w == 0) return;
    float m = -INFINITY, l = 0.f;
    for (int k = threadIdx.x & 31; k < meta.w; k += 32) m = fmaxf(m, a.part_ml[at(k)].x);
#pragma unroll
    for (int x = 16; x; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](const float2 ml, const float4 o) {
        const float w = ml.x == -INFINITY ? 0.f : ex2(ml.x - m);
        l = fmaf(w, ml.y, l);
        acc.x = fmaf(w, o.x, acc.x); acc.y = fmaf(w, o.y, acc.y); acc.z = fmaf(w, o.z, acc.z); acc.w = fmaf(w, o.w, acc.w);
    };
    if (u < meta.w) add(ml0, o0);
#pragma unroll 4
    for (int k = u + U; k < meta.w; k += U) add(a.part_ml[at(k)], a.part_o[at(k) * C + col]);
    sum_o[u][col] = acc;
    if (col == 0) sum_l[u] = l;
    __syncthreads();
    if (u != 0) return;
#pragma unroll
    for (int x = 1; x < U; ++x) {
        const float4 o = sum_o[x][col];
        acc.x += o.x; acc.y += o.y; acc.z += o.z; acc.w += o.w;
        l += sum_l[x];
    }
    const int i = r / a.pack, h = meta.y * a.pack + r % a.pack;
    const float inv = m == -INFINITY ? 0.f : 1.f / l;
    if (col * 4 < a.d)
        *reinterpret_cast<uint2*>(reinterpret_cast<T16*>(a.o) + meta.x * a.o_sb + i * a.o_sn + h * a.o_sh + col * 4) =
            make_uint2(pack2<BF16>(acc.x * inv, acc.y * inv), pack2<BF16>(acc.z * inv, acc.w * inv));
    if (col == 0) a.lse[((int64_t)meta.x * a.H + h) * a.Nq + i] = kLn2 * ((m - kPShift) + log2f(l));
}
