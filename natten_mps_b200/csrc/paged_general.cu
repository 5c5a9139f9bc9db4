// Attention over a paged cache for any head dim up to 256, any strides and every type but float64, in float32 arithmetic on the
// FMA pipe.  It serves float32, and 16-bit calls that the tensor-core kernels do not take.
//
// A tile is 16 rows by 32 keys.  Keys and values are fetched through the page table into shared memory as float32, a tile ahead of
// the products (float32 rows on 16-byte boundaries asynchronously).  Each of the four warps holds four rows: a lane forms the scores
// of one key (the key's row from its own padded line of shared memory, the query's broadcast), the softmax runs over the lanes
// with a running maximum, and for the weighted sum a lane holds four channels of every 128 of the four rows; with fewer than 128
// channels groups of lanes take different keys.
//
// What bounds a small call is latency: with one row fetched at a time, a chunk of 130 tokens over 1021 (2 sequences, 4 heads of 32
// on 2) took 55 us, with a tile fetched ahead 27.
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

// Rows r0, r0 + at_once, ... below `rows` of a tile: line r of `pitch` floats from src + place(r), zero where that is negative
// (and past D).  A row's chunks are spread over `across` lanes (a power of two).
template <typename T, int VEC, typename Place>
__device__ __forceinline__ void fetch_rows(float* dst, int pitch, const T* src, int rows, int D, int padded, int across, int warp, int warps, int lane,
                                           Place&& place)
{
    const int at_once = 32 / across, c0 = (lane & (across - 1)) * VEC, sub = lane / across;
    if constexpr (sizeof(T) == 4 && VEC == 4) {
        for (int r = warp * at_once; r < rows; r += warps * at_once) {
            const long long o = place(r + sub);              // (a shuffle: all lanes)
            for (int c = c0; c < padded; c += across * VEC) {
                const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(dst + (r + sub) * pitch + c));
                const int n = o >= 0 ? 16 : 0;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(o >= 0 ? src + o + c : src), "r"(n) : "memory");
            }
        }
    } else {
        constexpr int kBatch = 4;
        for (int block = 0; block < padded; block += across * VEC) {
            const int c = block + c0;
            for (int r = warp * at_once; r < rows; r += kBatch * warps * at_once) {
                Vec<T, VEC> x[kBatch];
                bool there[kBatch];
#pragma unroll
                for (int j = 0; j < kBatch; ++j) {
                    const int k = r + j * warps * at_once;
                    const long long o = place(k < rows ? k + sub : 0);
                    there[j] = k < rows && o >= 0 && c < D;  // D is a multiple of VEC
                    if (there[j]) x[j] = *reinterpret_cast<const Vec<T, VEC>*>(src + o + c);
                }
#pragma unroll
                for (int j = 0; j < kBatch; ++j) {
                    const int k = r + j * warps * at_once;
                    if (k >= rows) break;
#pragma unroll
                    for (int i = 0; i < VEC; ++i)
                        if (c + i < padded) dst[(k + sub) * pitch + c + i] = there[j] ? to_float(x[j].x[i]) : 0.f;
                }
            }
        }
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
    float *Q = shared_floats, *tiles = Q + kRows * pitch;    // two tiles of keys and values
    int across = 2;                          // (two rows' halves at least: 16 rows at a time at most)
    while (across < 32 && across * VEC < padded) across *= 2;
    int wide = 1;                            // lanes that share a row's channels in the weighted sum; 32 / wide groups take different keys
    while (wide < 32 && wide * 4 < padded) wide *= 2;
    const int group = lane / wide, groups = 32 / wide, channel = 4 * (lane & (wide - 1));
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
        __syncthreads();                     // the last unit's tiles have been read
        fetch_rows<T, VEC>(Q, pitch, q, kRows, A.D, padded, across, warp, kThreads / 32, lane,
                           [&](int r) { return r < x.rows ? query_offset(A, x, p.h, r) : -1ll; });
        unsigned seen_next = 0u;
        int page = 0, slot = 0;
        bool there = p.work && locate(A, x, x.base + p.x0 * kKeys + lane, page, slot);       // lane's key of the next tile to fetch
        auto fetch_tile = [&](int j) {
            float *Kt = tiles + (j & 1) * 2 * kKeys * pitch, *Vt = Kt + kKeys * pitch;
            const long long ko = there ? page * A.ks[0] + slot * A.ks[1] + p.h * A.ks[2] : -1,
                            vo = there ? page * A.vs[0] + slot * A.vs[1] + p.h * A.vs[2] : -1;
            seen_next = __ballot_sync(0xffffffffu, there);
            there = j + 1 < p.x1 && locate(A, x, x.base + (j + 1) * kKeys + lane, page, slot);
            fetch_rows<T, VEC>(Kt, pitch, kc, kKeys, A.D, padded, across, warp, kThreads / 32, lane,
                               [&](int r) { return __shfl_sync(0xffffffffu, ko, r); });
            fetch_rows<T, VEC>(Vt, pitch, vc, kKeys, A.D, padded, across, warp, kThreads / 32, lane,
                               [&](int r) { return __shfl_sync(0xffffffffu, vo, r); });
        };
        if (p.work) fetch_tile(p.x0);
        asm volatile("cp.async.commit_group;" ::: "memory");

        for (int j = p.x0; j < p.x1; ++j) {
            const int base = x.base + j * kKeys;
            const unsigned seen = seen_next;
            if (j + 1 < p.x1) fetch_tile(j + 1);
            asm volatile("cp.async.commit_group;" ::: "memory");
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            __syncthreads();                 // tile j is there
            const float *Kt = tiles + (j & 1) * 2 * kKeys * pitch, *Vt = Kt + kKeys * pitch;

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
                for (int k = group; k < kKeys; k += groups) {
                    float w[kPerWarp];
#pragma unroll
                    for (int r = 0; r < kPerWarp; ++r) w[r] = weights[warp * kPerWarp + r][k];
#pragma unroll
                    for (int c = 0; c < DC; ++c) {
                        const int d = 128 * c + channel;
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
            __syncthreads();                 // tile j has been read
        }
        for (int o = wide; o < 32; o *= 2)   // the groups' sums
#pragma unroll
            for (int r = 0; r < kPerWarp; ++r)
#pragma unroll
                for (int c = 0; c < DC; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[r][c][e] += __shfl_xor_sync(0xffffffffu, acc[r][c][e], o);

        const bool direct = clear || p.whole;
        const int where = 2 * (int)blockIdx.x + (p.x0 == 0 ? 1 : 0);
        if (!direct && p.x0 == 0) told = {piece.column * A.Hkv + p.h, piece.parts(A, blockIdx.x)};
#pragma unroll
        for (int r = 0; r < kPerWarp; ++r) {
            const int row = warp * kPerWarp + r;
            if (row >= x.rows) continue;
            const float inv = direct ? (l[r] > 0.f ? 1.f / l[r] : l[r]) : 1.f;          // a NaN stays one
            if (direct && lane == 0 && A.lse)
                A.lse[index[r]] = l[r] == 0.f ? -CUDART_INF_F : (m[r] + log2f(l[r])) * 0.6931471805599453f;
            if (!direct && lane == 0) slot_sums(A, where)[row] = make_float2(m[r], l[r]);
#pragma unroll
            for (int c = 0; c < DC; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int d = 128 * c + channel + e;
                    if (d >= A.D || group != 0) continue;
                    if (direct) static_cast<T*>(A.out)[index[r] * A.D + d] = from_float<T>(acc[r][c][e] * inv);
                    else slot_out(A, where)[row * A.D + d] = acc[r][c][e];
                }
        }
    }
    if (tid == 0 && !A.whole) reinterpret_cast<Shared*>(A.ws)[blockIdx.x] = told;
}

} // namespace

bool general_shape(int dtype, const Args& A, Shape& shape)
{
    if (dtype != NATTEN_F32 && dtype != NATTEN_F16 && dtype != NATTEN_BF16) return false;
    shape = {kRows, kKeys, 1, 1, 16, 3 * sm_count()};
    return A.D <= 256;
}

int general_run(int dtype, const Args& A, bool aligned, cudaStream_t s)
{
    const int pitch = ((A.D + 3) & ~3) + 4, smem = (kRows + 4 * kKeys) * pitch * (int)sizeof(float);
    cudaError_t err = cudaSuccess;
    auto go = [&](auto type, auto vec, auto dc) {
        auto* kernel = general_kernel<decltype(type), decltype(vec)::value, decltype(dc)::value>;
        err = ensure_dynamic_smem((const void*)kernel, (kRows + 4 * kKeys) * 260 * (int)sizeof(float));
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
