// Attention over a paged cache for few rows a unit (decoding steps, a few proposed tokens), 16-bit types: warp-level matrix
// products, each warp on its own keys.
//
// Such calls are bound by reading the cache: with 16 rows a key of 128 channels is 512 bytes against 8 Kflop.  So a CTA's
// eight warps (four above 128 channels) share a unit's rows and split its keys: of a tile of 8 * NK keys a warp fetches NK of its own (asynchronous 16-byte
// copies, kStages - 1 steps ahead, rows found through the page table one step before that), multiplies, runs its own softmax with
// its own maximum, and accumulates all channels of its weighted sum in registers.  Nothing in the loop waits for another warp.
// At the end of the unit the warps' partial results are joined through shared memory.
//
// Measured on one B200, bf16, 16 heads of 128 on 4: one token for each of 64 sequences of 2048 - 16384 tokens 191 us in a graph,
// 192 - 205 us over ten runs with other inputs in between (5.9 - 6.4 TB/s with the join, 90 - 97 % of a copy); 8 sequences through a window of 255 7.7 us, where lengths, page table, first keys and the join of the warps
// follow each other.  Eight warps a CTA or four and two CTAs an SM: with more short units than SMs two CTAs fill each other's
// beginnings and ends (128 sequences, window 512: 31 us against 37.5), with fewer the unit's keys want all warps (32 sequences of
// 512: 10.4 against 14.3).
//
// Weights are rounded to the tensors' type for their product with the values, which takes one type: half a step of each, as much as
// the rounding of the output; the row sum adds them as they were.  Against 64 bits the outputs are off by 0.0020 - 0.0022 of their size
// in bfloat16 and 0.00027 in float16, where the output's rounding alone leaves 0.0017 and 0.00021.
//
// A key that no row of the unit sees (behind the last query, in front of the first window, on a page that is not there) is not
// fetched: its line of shared memory is zero.  One that some rows see and others do not is multiplied by a weight of zero in those,
// so there a NaN or Inf value reaches them, too.
#include "../../include/natten_b200.h"

#include "device_cache.cuh"
#include "paged.cuh"
#include "simt_kernels.cuh"
#include "tc_common.cuh"
#include "tc_plan.cuh"
#include "warp_mma.cuh"

#include <math_constants.h>

#include <type_traits>

namespace natten {
namespace paged {

using tc::smem_u32;
using tcplan::cvt_pack;
using tcplan::fast_exp2;

namespace {

// MT: tiles of 16 rows; DP: head dim rounded up to 32, 64, 128 or 256; NW: warps of a CTA
template <int DP, int MT, int NW> struct Cfg {
    static constexpr int kWarps = NW, kThreads = 32 * kWarps, kPerSm = DP == 256 ? 1 : 8 / NW;
    static constexpr int kKeys = DP <= 64 ? 32 : 16;             // keys of a warp's step
    static constexpr int kStages = 3;
    static constexpr int kRowBytes = DP * 2, kChunks = DP / 8;   // 16-byte chunks of a row
    static constexpr int kTile = kKeys * kRowBytes;              // K (or V) of a step
    static constexpr int kWarpBytes = kStages * 2 * kTile;
    static constexpr int kRows = 16 * MT;
    static constexpr int kQ = kRows * kRowBytes;
    static constexpr int kPitch = DP + 4;                        // floats of a row of the exchange (over the stages)
    static constexpr int kExchange = kWarps * kRows * kPitch * 4;
    static constexpr int kStageBytes = kWarps * kWarpBytes > kExchange ? kWarps * kWarpBytes : kExchange;
    static constexpr int kSums = kQ + kStageBytes;               // float2 [kWarps][kRows], unsigned [kWarps][kStages], scratch
    static constexpr int kSmem = kSums + kWarps * kRows * 8 + kWarps * kStages * 4 + 16 + (int)sizeof(Piece::Scratch);
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there)
{
    const int n = there ? 16 : 0;            // 0: nothing is read, the chunk is zero
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// chunk c of row r: eight rows' equal chunks lie in different banks
template <int DP> __device__ __forceinline__ uint32_t at(int r, int c)
{
    return r * (DP * 2) + ((DP >= 64 ? c ^ (r & 7) : c ^ ((r >> 1) & 3)) << 4);
}

template <int DP, int MT, int NW, bool BF16>
__global__ void __launch_bounds__(Cfg<DP, MT, NW>::kThreads, Cfg<DP, MT, NW>::kPerSm) warp_kernel(const __grid_constant__ Args A)
{
    using C = Cfg<DP, MT, NW>;
    constexpr int NK = C::kKeys, NT = NK / 8, ST = C::kStages, kWarps = C::kWarps, kThreads = C::kThreads;
    extern __shared__ __align__(128) unsigned char smem[];
    float2* sums = reinterpret_cast<float2*>(smem + C::kSums);
    volatile unsigned* there_words = reinterpret_cast<unsigned*>(smem + C::kSums + kWarps * C::kRows * 8);
    Piece::Scratch* scratch = reinterpret_cast<Piece::Scratch*>(smem + C::kSums + kWarps * C::kRows * 8 + ((kWarps * ST * 4 + 15) & ~15));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t q_base = smem_u32(smem), stage_base = q_base + C::kQ + warp * C::kWarpBytes;
    const uint16_t *q = static_cast<const uint16_t*>(A.q), *kc = static_cast<const uint16_t*>(A.kc), *vc = static_cast<const uint16_t*>(A.vc);
    const int mi = lane >> 3, mr = lane & 7;                     // matrix and row that this lane addresses for ldmatrix

    Piece piece;
    piece.begin<kThreads>(A, blockIdx.x, scratch);
    let_dependents_launch();
    Shared told{-1, 0};
    for (; piece.more(); piece.advance(A)) {
        const Piece::Portion p = piece.portion(A);
        const Tile& x = piece.tile;
        const bool clear = x.n == 0 && p.first;
        if (!p.work && !clear) continue;

        const int steps = p.x1 - p.x0, first_key = x.lo + p.x0 * (kWarps * NK) + warp * NK;
        // ---- fetching ----
        struct Place { int page, slot; bool there; };
        auto look_up = [&](int step) {       // lane's key of the step: its place in the cache
            Place y{0, 0, false};
            y.there = step < steps && lane < NK && locate(A, x, first_key + step * (kWarps * NK) + lane, y.page, y.slot);
            return y;
        };
        auto fetch = [&](int step, const Place& y) {
            const int page = y.page, slot = y.slot;
            const bool there = y.there;
            if (step < steps) {
                const unsigned seen = __ballot_sync(0xffffffffu, there);
                const int s = step % ST;
                if (lane == 0) there_words[warp * ST + s] = seen;
                const long long ko = there ? page * A.ks[0] + slot * A.ks[1] + p.h * A.ks[2] : 0,
                                vo = there ? page * A.vs[0] + slot * A.vs[1] + p.h * A.vs[2] : 0;
                const uint32_t k_dst = stage_base + s * 2 * C::kTile, v_dst = k_dst + C::kTile;
                constexpr int kLanes = C::kChunks < 32 ? C::kChunks : 32, kAtOnce = 32 / kLanes;   // lanes of a row, rows at a time
                const int c = lane % kLanes;
                const bool real = c * 8 < A.D;
#pragma unroll
                for (int i = 0; i < NK; i += kAtOnce) {
                    const int r = i + lane / kLanes;
                    const long long kr = __shfl_sync(0xffffffffu, ko, r), vr = __shfl_sync(0xffffffffu, vo, r);
                    const bool here = real && ((seen >> r) & 1u);
                    copy16(k_dst + at<DP>(r, c), here ? kc + kr + c * 8 : q, here);
                    copy16(v_dst + at<DP>(r, c), here ? vc + vr + c * 8 : q, here);
                }
            }
            copies_commit();
        };

        // ---- the unit's queries ----
        Place ahead[ST];                     // of the first steps, all asked for at once; then ahead[0]: of the next step to fetch
#pragma unroll
        for (int s = 0; s < ST; ++s) ahead[s] = look_up(s);
        for (int e = tid; e < C::kRows * C::kChunks; e += kThreads) {
            const int r = e / C::kChunks, c = e % C::kChunks;
            const bool here = r < x.rows && c * 8 < A.D;
            copy16(q_base + at<DP>(r, c), here ? q + query_offset(A, x, p.h, r) + c * 8 : q, here);
        }
        copies_commit();
#pragma unroll
        for (int s = 0; s < ST - 1; ++s) fetch(s, ahead[s]);
        ahead[0] = ahead[ST - 1];
        int tq[MT][2], t_least = 0x7fffffff, t_most = -1;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = 16 * m + 8 * i + (lane >> 2);
                long long index;
                tq[m][i] = -1;
                if (r < x.rows && row_of(A, x, p.h, r, index, tq[m][i])) {
                    t_least = min(t_least, tq[m][i]);
                    t_most = max(t_most, tq[m][i]);
                } else {
                    tq[m][i] = -1;           // sees nothing
                }
            }
        t_least = __reduce_min_sync(0xffffffffu, t_least);
        t_most = __reduce_max_sync(0xffffffffu, t_most);
        copies_wait<ST - 1>();
        __syncthreads();
        uint32_t qf[MT][DP / 16][4];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int k = 0; k < DP / 16; ++k)
                wmma16::ldsm_x4(qf[m][k], q_base + at<DP>(16 * m + (mi & 1) * 8 + mr, 2 * k + (mi >> 1)));

        float top[MT][2], total[MT][2], acc[MT][DP / 8][4];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            top[m][0] = top[m][1] = -CUDART_INF_F;
            total[m][0] = total[m][1] = 0.f;
#pragma unroll
            for (int n = 0; n < DP / 8; ++n) acc[m][n][0] = acc[m][n][1] = acc[m][n][2] = acc[m][n][3] = 0.f;
        }

        for (int step = 0; step < steps; ++step) {
            copies_wait<ST - 2>();
            __syncwarp();                    // every lane's copies of this step have landed, and the last step's buffers have been read
            fetch(step + ST - 1, ahead[0]);
            ahead[0] = look_up(step + ST);
            const int s = step % ST, base = first_key + step * (kWarps * NK);
            const unsigned seen = there_words[warp * ST + s];
            if (seen == 0u) continue;
            const uint32_t k_src = stage_base + s * 2 * C::kTile, v_src = k_src + C::kTile;
            // two sums a score (even and odd steps along the channels): half the chain of dependent products
            float sc[MT][NT][4], odd[MT][NT][4];
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sc[m][n][e] = odd[m][n][e] = 0.f;
#pragma unroll
            for (int k = 0; k < DP / 16; ++k)
#pragma unroll
                for (int n = 0; n < NT; n += 2) {
                    uint32_t b[4];
                    wmma16::ldsm_x4(b, k_src + at<DP>(8 * n + (mi >> 1) * 8 + mr, 2 * k + (mi & 1)));
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        wmma16::mma_16816<BF16>(k & 1 ? odd[m][n] : sc[m][n], qf[m][k], b[0], b[1]);
                        wmma16::mma_16816<BF16>(k & 1 ? odd[m][n + 1] : sc[m][n + 1], qf[m][k], b[2], b[3]);
                    }
                }
            const unsigned every = NK == 32 ? 0xffffffffu : (1u << NK) - 1u;
            const bool open = seen == every && base + NK - 1 <= t_least && t_most - base < A.K;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float v = (sc[m][n][e] + odd[m][n][e]) * A.scale_log2;
                        if (!open) {
                            const int j = 8 * n + 2 * (lane & 3) + (e & 1), t = base + j, to = tq[m][e >> 1];
                            if (!(((seen >> j) & 1u) && t <= to && to - t < A.K)) v = -CUDART_INF_F;
                        }
                        sc[m][n][e] = v;
                    }
            uint32_t w[MT][NT][2];
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float now = top[m][i];
#pragma unroll
                    for (int n = 0; n < NT; ++n) now = fmaxf(now, fmaxf(sc[m][n][2 * i], sc[m][n][2 * i + 1]));
                    now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, 1));
                    now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, 2));
                    const float base_m = now == -CUDART_INF_F ? 0.f : now;
                    if (__any_sync(0xffffffffu, now > top[m][i])) {
                        const float f = fast_exp2(top[m][i] - base_m);
                        total[m][i] *= f;
#pragma unroll
                        for (int n = 0; n < DP / 8; ++n) {
                            acc[m][n][2 * i] *= f;
                            acc[m][n][2 * i + 1] *= f;
                        }
                        top[m][i] = now;
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const float a = fast_exp2(sc[m][n][2 * i] - base_m), b = fast_exp2(sc[m][n][2 * i + 1] - base_m);
                        total[m][i] += a + b;
                        w[m][n][i] = cvt_pack<BF16>(a, b);       // weights are at most 1: half a step of the type
                    }
                }
#pragma unroll
            for (int k = 0; k < NK / 16; ++k)
#pragma unroll
                for (int n = 0; n < DP / 8; n += 2) {
                    uint32_t b[4];
                    wmma16::ldsm_x4_t(b, v_src + at<DP>(16 * k + (mi & 1) * 8 + mr, n + (mi >> 1)));
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        const uint32_t a[4] = {w[m][2 * k][0], w[m][2 * k][1], w[m][2 * k + 1][0], w[m][2 * k + 1][1]};
                        wmma16::mma_16816<BF16>(acc[m][n], a, b[0], b[1]);
                        wmma16::mma_16816<BF16>(acc[m][n + 1], a, b[2], b[3]);
                    }
                }
        }

        // ---- join the warps ----
        copies_wait<0>();
        __syncthreads();                     // the stages are free
        float* exchange = reinterpret_cast<float*>(smem + C::kQ);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = 16 * m + 8 * i + (lane >> 2);
                float l = total[m][i];
                l += __shfl_xor_sync(0xffffffffu, l, 1);
                l += __shfl_xor_sync(0xffffffffu, l, 2);
                if (r >= x.rows) continue;
                if ((lane & 3) == 0) sums[warp * C::kRows + r] = make_float2(top[m][i], l);
                float* line = exchange + (warp * C::kRows + r) * C::kPitch + 2 * (lane & 3);
#pragma unroll
                for (int n = 0; n < DP / 8; ++n) *reinterpret_cast<float2*>(line + 8 * n) = make_float2(acc[m][n][2 * i], acc[m][n][2 * i + 1]);
            }
        __syncthreads();
        const bool direct = clear || p.whole;
        const int where = 2 * (int)blockIdx.x + (p.x0 == 0 ? 1 : 0);
        if (!direct && p.x0 == 0) told = {piece.column * A.Hkv + p.h, piece.parts(A, blockIdx.x)};
        for (int e = tid; e < x.rows * C::kChunks; e += kThreads) {
            const int r = e / C::kChunks, c = e % C::kChunks;
            if (8 * c >= A.D) continue;
            float m = -CUDART_INF_F, l = 0.f, f[kWarps], o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < kWarps; ++k) m = fmaxf(m, sums[k * C::kRows + r].x);
            const float base_m = m == -CUDART_INF_F ? 0.f : m;
#pragma unroll
            for (int k = 0; k < kWarps; ++k) {
                const float2 s = sums[k * C::kRows + r];
                f[k] = fast_exp2(s.x - base_m);
                l = fmaf(f[k], s.y, l);
                const float4* y = reinterpret_cast<const float4*>(exchange + (k * C::kRows + r) * C::kPitch + 8 * c);
                const float4 a = y[0], b = y[1];
                o[0] = fmaf(f[k], a.x, o[0]); o[1] = fmaf(f[k], a.y, o[1]); o[2] = fmaf(f[k], a.z, o[2]); o[3] = fmaf(f[k], a.w, o[3]);
                o[4] = fmaf(f[k], b.x, o[4]); o[5] = fmaf(f[k], b.y, o[5]); o[6] = fmaf(f[k], b.z, o[6]); o[7] = fmaf(f[k], b.w, o[7]);
            }
            if (direct) {
                long long index;
                int t;
                const bool live = row_of(A, x, p.h, r, index, t);
                const float inv = !live ? 0.f : l > 0.f ? 1.f / l : l;   // a NaN stays one
                const bool none = !live || l == 0.f;
                uint4 y = make_uint4(0u, 0u, 0u, 0u);
                if (!none) {
                    y.x = cvt_pack<BF16>(o[0] * inv, o[1] * inv);
                    y.y = cvt_pack<BF16>(o[2] * inv, o[3] * inv);
                    y.z = cvt_pack<BF16>(o[4] * inv, o[5] * inv);
                    y.w = cvt_pack<BF16>(o[6] * inv, o[7] * inv);
                }
                reinterpret_cast<uint4*>(static_cast<uint16_t*>(A.out) + index * A.D)[c] = y;
                if (c == 0 && A.lse) A.lse[index] = none ? -CUDART_INF_F : (m + log2f(l)) * 0.6931471805599453f;
            } else {
                float4* y = reinterpret_cast<float4*>(slot_out(A, where) + (long long)r * A.D + 8 * c);
                y[0] = make_float4(o[0], o[1], o[2], o[3]);
                y[1] = make_float4(o[4], o[5], o[6], o[7]);
                if (c == 0) slot_sums(A, where)[r] = make_float2(m, l);
            }
        }
        __syncthreads();                     // the exchange has been read
    }
    if (tid == 0 && !A.whole) reinterpret_cast<Shared*>(A.ws)[blockIdx.x] = told;
}

// f(DP, MT, NW) for the call's head dim, rows of a tile and warps of a CTA
template <typename F> auto by_config(const Args& A, int M, int warps, F&& f)
{
    auto by_warps = [&](auto dp, auto mt) {
        constexpr int kDim = decltype(dp)::value;
        if constexpr (kDim < 256) {
            if (warps == 8) return f(dp, mt, std::integral_constant<int, 8>{});
        }
        return f(dp, mt, std::integral_constant<int, 4>{});
    };
    auto by_rows = [&](auto dp) {
        constexpr int kDim = decltype(dp)::value;
        if constexpr (kDim < 256) {
            if (M == 32) return by_warps(dp, std::integral_constant<int, 2>{});
        }
        return by_warps(dp, std::integral_constant<int, 1>{});
    };
    if (A.D <= 32) return by_rows(std::integral_constant<int, 32>{});
    if (A.D <= 64) return by_rows(std::integral_constant<int, 64>{});
    if (A.D <= 128) return by_rows(std::integral_constant<int, 128>{});
    return by_rows(std::integral_constant<int, 256>{});
}

} // namespace

// `warps`: 8 (one CTA an SM) or 4 (two).
bool warp_shape(int dtype, const Args& A, bool aligned, int warps, Shape& shape)
{
    if ((dtype != NATTEN_F16 && dtype != NATTEN_BF16) || !aligned || A.D > 256) return false;
    // 16 rows, or 32 where a class has more (256 channels of 32 rows do not fit the registers)
    const long long rows = ((long long)A.L + A.dil - 1) / A.dil * A.G;
    shape.M = rows > 16 && A.D <= 128 ? 32 : 16;
    by_config(A, shape.M, warps, [&](auto dp, auto mt, auto nw) {
        using C = Cfg<decltype(dp)::value, decltype(mt)::value, decltype(nw)::value>;
        shape.keys = C::kWarps * C::kKeys;
        shape.ctas = C::kPerSm * sm_count();
        shape.most = 64 / C::kWarps;
    });
    shape.overhead = 1;
    shape.least = 2;
    return true;
}

int warp_run(int dtype, const Args& A, int warps, cudaStream_t s)
{
    return by_config(A, A.M, warps, [&](auto dp, auto mt, auto nw) {
        using C = Cfg<decltype(dp)::value, decltype(mt)::value, decltype(nw)::value>;
        cudaError_t err;
        auto go = [&](auto* kernel) {
            err = ensure_dynamic_smem((const void*)kernel, C::kSmem);
            if (err == cudaSuccess) kernel<<<A.ctas, C::kThreads, C::kSmem, s>>>(A);
        };
        if (dtype == NATTEN_BF16) go(warp_kernel<decltype(dp)::value, decltype(mt)::value, decltype(nw)::value, true>);
        else go(warp_kernel<decltype(dp)::value, decltype(mt)::value, decltype(nw)::value, false>);
        if (err == cudaSuccess) err = cudaGetLastError();
        simt_count_launch(1);
        return (int)err;
    });
}

} // namespace paged
} // namespace natten
