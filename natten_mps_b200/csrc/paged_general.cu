// Attention over a paged cache for any head dim up to 256, any strides and every type but float64, in float32 arithmetic on the
// FMA pipe.  It serves float32, and 16-bit calls that the tensor-core kernels do not take.
//
// A tile is 16 rows by 32 keys.  Keys and values are fetched through the page table into shared memory as float32.  Each of the
// four warps holds four rows: a lane forms the scores of one key (the key's row from its own padded line of shared memory, the
// query's broadcast), the softmax runs over the lanes with a running maximum, and for the weighted sum a lane holds four channels
// of every 128 of the four rows.
//
// A key that is masked for a row does not reach it, whatever it holds (NaN and Inf included).
#include "../../include/natten_b200.h"

#include "device_cache.cuh"
#include "paged.cuh"
#include "simt_kernels.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include <type_traits>

namespace natten {
namespace paged {
namespace {

constexpr int kThreads = 128, kRows = 16, kKeys = 32, kPerWarp = 4;

template <typename T> __device__ __forceinline__ float to_float(T x);
template <> __device__ __forceinline__ float to_float(float x) { return x; }
template <> __device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float(float x) { return x; }
template <> __device__ __forceinline__ __half from_float(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float x) { return __float2bfloat16_rn(x); }

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Vec { T x[VEC]; };

// one row of global memory into a line of `pitch` floats; channels past D are zero.  `lanes` threads share it.
template <typename T, int VEC>
__device__ __forceinline__ void fetch_row(float* dst, const T* src, bool there, int D, int padded, int lane, int lanes)
{
    for (int c = lane * VEC; c < padded; c += lanes * VEC) {
        float x[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) x[i] = 0.f;
        if (there && c < D) {                // D is a multiple of VEC
            const Vec<T, VEC> y = *reinterpret_cast<const Vec<T, VEC>*>(src + c);
#pragma unroll
            for (int i = 0; i < VEC; ++i) x[i] = to_float(y.x[i]);
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (c + i < padded) dst[c + i] = x[i];
    }
}

// DC: groups of 128 channels
template <typename T, int VEC, int DC>
__global__ void __launch_bounds__(kThreads) general_kernel(const __grid_constant__ Args A)
{
    extern __shared__ __align__(16) float shared_floats[];
    __shared__ Piece::Scratch scratch;
    __shared__ float weights[kRows][kKeys];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int padded = (A.D + 3) & ~3, pitch = padded + 4;
    float *Q = shared_floats, *Kt = Q + kRows * pitch, *Vt = Kt + kKeys * pitch;
    const T *q = static_cast<const T*>(A.q), *kc = static_cast<const T*>(A.kc), *vc = static_cast<const T*>(A.vc);

    Piece piece;
    piece.begin<kThreads>(A, blockIdx.x, &scratch);
    let_dependents_launch();
    Shared told{-1, 0};
    for (; piece.more(); piece.advance(A)) {
        const Piece::Portion p = piece.portion(A);
        const Tile& x = piece.tile;
        const bool clear = x.n == 0 && p.first;
        if (!p.work && !clear) continue;

        float m[kPerWarp], l[kPerWarp], acc[kPerWarp][DC][4];
        int tq[kPerWarp];
#pragma unroll
        for (int r = 0; r < kPerWarp; ++r) {
            m[r] = -CUDART_INF_F;
            l[r] = 0.f;
#pragma unroll
            for (int c = 0; c < DC; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[r][c][e] = 0.f;
        }
        long long index[kPerWarp];
        bool live[kPerWarp];
#pragma unroll
        for (int r = 0; r < kPerWarp; ++r) {
            const int row = warp * kPerWarp + r;
            index[r] = -1;
            tq[r] = -1;
            live[r] = false;
            if (row < x.rows) live[r] = row_of(A, x, p.h, row, index[r], tq[r]);
        }
        __syncthreads();
        for (int r = warp; r < kRows; r += kThreads / 32)
            fetch_row<T, VEC>(Q + r * pitch, r < x.rows ? q + query_offset(A, x, p.h, r) : nullptr, r < x.rows, A.D, padded, lane, 32);

        for (int j = p.x0; j < p.x1; ++j) {
            const int base = x.lo + j * kKeys;
            __syncthreads();                 // the previous tile has been read
            int page = 0, slot = 0;
            const bool there = locate(A, x, base + lane, page, slot);
            const unsigned seen = __ballot_sync(0xffffffffu, there);
            const long long ko = page * A.ks[0] + slot * A.ks[1] + p.h * A.ks[2], vo = page * A.vs[0] + slot * A.vs[1] + p.h * A.vs[2];
            for (int r = warp; r < kKeys; r += kThreads / 32) {
                const long long kr = __shfl_sync(0xffffffffu, ko, r), vr = __shfl_sync(0xffffffffu, vo, r);
                const bool here = (seen >> r) & 1u;
                fetch_row<T, VEC>(Kt + r * pitch, here ? kc + kr : nullptr, here, A.D, padded, lane, 32);
                fetch_row<T, VEC>(Vt + r * pitch, here ? vc + vr : nullptr, here, A.D, padded, lane, 32);
            }
            __syncthreads();

            float s[kPerWarp] = {0.f, 0.f, 0.f, 0.f};
            const float4* k4 = reinterpret_cast<const float4*>(Kt + lane * pitch);
            const float4* q4 = reinterpret_cast<const float4*>(Q + warp * kPerWarp * pitch);
            for (int c = 0; c < padded / 4; ++c) {
                const float4 k = k4[c];
#pragma unroll
                for (int r = 0; r < kPerWarp; ++r) {
                    const float4 y = q4[r * (pitch / 4) + c];
                    s[r] = fmaf(k.x, y.x, fmaf(k.y, y.y, fmaf(k.z, y.z, fmaf(k.w, y.w, s[r]))));
                }
            }
            const int t = base + lane;
            bool masked = false;
#pragma unroll
            for (int r = 0; r < kPerWarp; ++r) {
                const bool ok = ((seen >> lane) & 1u) && live[r] && t <= tq[r] && tq[r] - t < A.K;
                masked = masked || !ok;
                float v = ok ? s[r] * A.scale_log2 : -CUDART_INF_F, top = v;
#pragma unroll
                for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                const float now = fmaxf(m[r], top), base_m = now == -CUDART_INF_F ? 0.f : now;
                const float w = ok ? exp2f(v - base_m) : 0.f, f = exp2f(m[r] - base_m);
                float sum = w;
#pragma unroll
                for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                m[r] = now;
                l[r] = l[r] * f + sum;
#pragma unroll
                for (int c = 0; c < DC; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[r][c][e] *= f;
                weights[warp * kPerWarp + r][lane] = w;
            }
            const bool any_masked = __any_sync(0xffffffffu, masked);
            __syncwarp();
            auto add = [&](auto selected) {
                for (int k = 0; k < kKeys; ++k) {
                    float w[kPerWarp];
#pragma unroll
                    for (int r = 0; r < kPerWarp; ++r) w[r] = weights[warp * kPerWarp + r][k];
#pragma unroll
                    for (int c = 0; c < DC; ++c) {
                        const int d = 128 * c + 4 * lane;
                        if (d >= padded) continue;
                        const float4 v = *reinterpret_cast<const float4*>(Vt + k * pitch + d);
#pragma unroll
                        for (int r = 0; r < kPerWarp; ++r) {
                            if (decltype(selected)::value && w[r] == 0.f) continue;
                            acc[r][c][0] = fmaf(w[r], v.x, acc[r][c][0]);
                            acc[r][c][1] = fmaf(w[r], v.y, acc[r][c][1]);
                            acc[r][c][2] = fmaf(w[r], v.z, acc[r][c][2]);
                            acc[r][c][3] = fmaf(w[r], v.w, acc[r][c][3]);
                        }
                    }
                }
            };
            if (any_masked) add(std::true_type{});
            else add(std::false_type{});
        }

        const bool direct = clear || p.whole;
        const int slot = 2 * (int)blockIdx.x + (p.x0 == 0 ? 1 : 0);
        if (!direct && p.x0 == 0) told = {piece.column * A.Hkv + p.h, piece.parts(A, blockIdx.x)};
#pragma unroll
        for (int r = 0; r < kPerWarp; ++r) {
            const int row = warp * kPerWarp + r;
            if (row >= x.rows) continue;
            const float inv = direct ? (l[r] > 0.f ? 1.f / l[r] : l[r]) : 1.f;          // a NaN stays one
            if (direct && lane == 0 && A.lse)
                A.lse[index[r]] = l[r] == 0.f ? -CUDART_INF_F : (m[r] + log2f(l[r])) * 0.6931471805599453f;
            if (!direct && lane == 0) slot_sums(A, slot)[row] = make_float2(m[r], l[r]);
#pragma unroll
            for (int c = 0; c < DC; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int d = 128 * c + 4 * lane + e;
                    if (d >= A.D) continue;
                    if (direct) static_cast<T*>(A.out)[index[r] * A.D + d] = from_float<T>(acc[r][c][e] * inv);
                    else slot_out(A, slot)[row * A.D + d] = acc[r][c][e];
                }
        }
    }
    if (tid == 0) reinterpret_cast<Shared*>(A.ws)[blockIdx.x] = told;
}

} // namespace

bool general_shape(int dtype, const Args& A, bool, Shape& shape)
{
    if (dtype != NATTEN_F32 && dtype != NATTEN_F16 && dtype != NATTEN_BF16) return false;
    shape = {kRows, kKeys, 1, 1, 16, 3 * sm_count()};
    return A.D <= 256;
}

int general_run(int dtype, const Args& A, bool aligned, cudaStream_t s)
{
    const int pitch = ((A.D + 3) & ~3) + 4, smem = (kRows + 2 * kKeys) * pitch * (int)sizeof(float);
    cudaError_t err = cudaSuccess;
    auto go = [&](auto type, auto vec, auto dc) {
        auto* kernel = general_kernel<decltype(type), decltype(vec)::value, decltype(dc)::value>;
        err = ensure_dynamic_smem((const void*)kernel, (kRows + 2 * kKeys) * 260 * (int)sizeof(float));
        if (err == cudaSuccess) kernel<<<A.ctas, kThreads, smem, s>>>(A);
    };
    auto by_dim = [&](auto type, auto vec) {
        if (A.D <= 128) go(type, vec, std::integral_constant<int, 1>{});
        else go(type, vec, std::integral_constant<int, 2>{});
    };
    auto by_width = [&](auto type) {
        if (aligned) by_dim(type, std::integral_constant<int, 16 / (int)sizeof(type)>{});
        else by_dim(type, std::integral_constant<int, 1>{});
    };
    if (dtype == NATTEN_F32) by_width(float{});
    else if (dtype == NATTEN_F16) by_width(__half{});
    else by_width(__nv_bfloat16{});
    if (err == cudaSuccess) err = cudaGetLastError();
    simt_count_launch(1);
    return (int)err;
}

} // namespace paged
} // namespace natten
