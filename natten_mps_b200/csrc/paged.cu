// C entry of the attention over a paged cache: checks, choice of the kernel, and the kernel that joins the partial results of
// units that several CTAs share (see paged.cuh).
#include "../../include/natten_b200.h"

#include "device_cache.cuh"
#include "paged.cuh"
#include "simt_kernels.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include <algorithm>
#include <type_traits>

namespace natten {
namespace paged {
namespace {

constexpr int kJoinWarps = 8, kJoinThreads = 32 * kJoinWarps;

template <typename T> __device__ __forceinline__ T rounded(float x);
template <> __device__ __forceinline__ float rounded(float x) { return x; }
template <> __device__ __forceinline__ __half rounded(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 rounded(float x) { return __float2bfloat16_rn(x); }

// Block (c, y): rows y * ROWS ... of the unit that CTA c began and others went on with.  With M = max m_i its rows are
// sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i over the parts i.  Warps take a row each; where a block has fewer rows than warps
// several share a row's parts.  A lane holds four channels of every 128, and asks for several parts at a time: what this costs is
// the latency of the workspace, so everything that does not depend on an answer is asked for at once.
template <typename T, int ROWS, int DC> __global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ Args A)
{
    constexpr int kShare = ROWS >= kJoinWarps ? 1 : kJoinWarps / ROWS;   // warps of a row
    constexpr int kAtOnce = 8 / DC;                                      // parts asked for at a time
    __shared__ float4 others[kJoinWarps][32 * DC];
    __shared__ float other_sums[kJoinWarps];
    const int c = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, share = warp % kShare;
    wait_for_primary();
    const Shared mine = reinterpret_cast<const Shared*>(A.ws)[c];
    if (mine.unit < 0) return;
    const int column = mine.unit / A.Hkv, h = mine.unit - column * A.Hkv, parts = mine.parts;
    const Tile x = tile_of(A, column);
    auto slot = [&](int i) { return i == 0 ? 2 * c + 1 : 2 * (c + i); };
    for (int r = warp / kShare; r < ROWS; r += kJoinWarps / kShare) {    // as many rounds in every warp of the block
        const int row = blockIdx.y * ROWS + r;
        const bool real = row < x.rows;
        float top = -CUDART_INF_F;
        bool bad = false;
        if (real)
            for (int i = lane; i < parts; i += 32) {
                const float m = slot_sums(A, slot(i))[row].x;
                bad = bad || m != m;
                top = fmaxf(top, m);
            }
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (__any_sync(0xffffffffu, bad)) top = CUDART_NAN_F;
        const float base = top == -CUDART_INF_F ? 0.f : top;
        float total = 0.f;
        float4 acc[DC];
#pragma unroll
        for (int d = 0; d < DC; ++d) acc[d] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (real)
            for (int i0 = share; i0 < parts; i0 += kShare * kAtOnce) {
                float2 ml[kAtOnce];
                float4 o[kAtOnce][DC];
#pragma unroll
                for (int k = 0; k < kAtOnce; ++k) {
                    const int i = i0 + k * kShare;
                    ml[k] = make_float2(-CUDART_INF_F, 0.f);
                    if (i >= parts) continue;
                    ml[k] = slot_sums(A, slot(i))[row];
                    const float* src = slot_out(A, slot(i)) + (long long)row * A.D;
#pragma unroll
                    for (int d = 0; d < DC; ++d) {
                        const int ch = 128 * d + 4 * lane;
                        o[k][d] = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (A.D % 4 == 0) {
                            if (ch < A.D) o[k][d] = *reinterpret_cast<const float4*>(src + ch);
                        } else {
                            if (ch < A.D) o[k][d].x = src[ch];
                            if (ch + 1 < A.D) o[k][d].y = src[ch + 1];
                            if (ch + 2 < A.D) o[k][d].z = src[ch + 2];
                            if (ch + 3 < A.D) o[k][d].w = src[ch + 3];
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < kAtOnce; ++k) {
                    const float f = exp2f(ml[k].x - base);
                    if (ml[k].y == 0.f) continue;                        // a part that saw nothing (NaN scores leave m = -inf, l = NaN)
                    total = fmaf(f, ml[k].y, total);
#pragma unroll
                    for (int d = 0; d < DC; ++d) {
                        acc[d].x = fmaf(f, o[k][d].x, acc[d].x);
                        acc[d].y = fmaf(f, o[k][d].y, acc[d].y);
                        acc[d].z = fmaf(f, o[k][d].z, acc[d].z);
                        acc[d].w = fmaf(f, o[k][d].w, acc[d].w);
                    }
                }
            }
        if constexpr (kShare > 1) {
            __syncthreads();                                             // the last round's have been read
#pragma unroll
            for (int d = 0; d < DC; ++d) others[warp][32 * d + lane] = acc[d];
            if (lane == 0) other_sums[warp] = total;
            __syncthreads();
            if (share == 0) {
#pragma unroll
                for (int k = 1; k < kShare; ++k) {
                    total += other_sums[warp + k];
#pragma unroll
                    for (int d = 0; d < DC; ++d) {
                        const float4 y = others[warp + k][32 * d + lane];
                        acc[d].x += y.x;
                        acc[d].y += y.y;
                        acc[d].z += y.z;
                        acc[d].w += y.w;
                    }
                }
            }
        }
        if (!real || share != 0) continue;
        long long index;
        int t;
        const bool live = row_of(A, x, h, row, index, t);
        const bool some = live && total != 0.f;                          // (a NaN stays one)
        const float inv = some ? 1.f / total : 0.f;
#pragma unroll
        for (int d = 0; d < DC; ++d) {
            const float y[4] = {acc[d].x, acc[d].y, acc[d].z, acc[d].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int ch = 128 * d + 4 * lane + e;
                if (ch < A.D) static_cast<T*>(A.out)[index * A.D + ch] = rounded<T>(some ? y[e] * inv : 0.f);
            }
        }
        if (A.lse && lane == 0) A.lse[index] = some ? (base + log2f(total)) * 0.6931471805599453f : -CUDART_INF_F;
    }
}

// The joining kernel starts while the last CTAs of the kernel in front of it are still at work, and waits for their results.
int join(int dtype, const Args& A, cudaStream_t s)
{
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.blockDim = dim3(kJoinThreads);
    cfg.stream = s;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    cudaError_t err = cudaSuccess;
    auto go = [&](auto type, auto rows, auto dc) {
        constexpr int kRows = decltype(rows)::value;
        cfg.gridDim = dim3(A.ctas, (A.M + kRows - 1) / kRows);
        err = cudaLaunchKernelEx(&cfg, join_kernel<decltype(type), kRows, decltype(dc)::value>, A);
    };
    // Many rows: a block for 32 of them.  Few rows may have a part in every CTA: two rows a block, four warps each (one sequence
    // of 65536 tokens and one key/value head: 18 us in all; a warp a row, part after part, 181).
    auto by_rows = [&](auto type, auto dc) {
        if (A.M > 32) go(type, std::integral_constant<int, 32>{}, dc);
        else go(type, std::integral_constant<int, 2>{}, dc);
    };
    auto by_dim = [&](auto type) {
        if (A.D <= 128) by_rows(type, std::integral_constant<int, 1>{});
        else by_rows(type, std::integral_constant<int, 2>{});
    };
    if (dtype == NATTEN_F32) by_dim(float{});
    else if (dtype == NATTEN_F16) by_dim(__half{});
    else by_dim(__nv_bfloat16{});
    simt_count_launch(1);
    return (int)err;
}

// Tile counts of the padded batch, whatever the lengths are.  False: more units than 31 bits number.
bool divide(Args& A, const Shape& shape)
{
    A.M = shape.M;
    A.keys = shape.keys;
    A.overhead = shape.overhead;
    A.least = shape.least;
    A.align = 1;
    // tiles that the keys of a unit can have: a window and the queries behind its first, what the table can hold
    const long long held = (long long)A.table_width * A.page_size / A.dil + 1;
    const long long reach = std::min(held, (long long)A.K + (A.M + A.G - 1) / A.G);
    A.whole = reach <= (long long)(shape.most - 1) * shape.keys;
    const int queries = A.L / A.dil;
    A.long_classes = A.L - queries * A.dil;
    auto tiles = [&](long long n) { return (n * A.G + A.M - 1) / A.M; };
    const long long a = tiles((long long)queries + 1), b = tiles(queries), short_classes = queries ? A.dil - A.long_classes : 0;
    const long long per = A.long_classes * a + short_classes * b;
    if (per * A.B * A.Hkv > 0x3fffffff || ((long long)queries + 1) * A.G > 0x3fffffff) return false;
    A.tiles_long = (int)a;
    A.tiles_short = (int)b;
    A.per_seq = (int)per;
    A.columns = (int)(per * A.B);
    A.ctas = shape.ctas;
    A.by_group = FastDiv((uint32_t)A.G);
    A.by_ctas = FastDiv((uint32_t)A.ctas);
    A.by_dil = FastDiv((uint32_t)A.dil);
    A.by_seq = FastDiv((uint32_t)std::max(1, A.per_seq));
    A.by_long = FastDiv((uint32_t)std::max(1, A.tiles_long));
    A.by_short = FastDiv((uint32_t)std::max(1, A.tiles_short));
    A.capacity = (int)std::min<long long>((long long)A.table_width * A.page_size, kAllOfThePast);
    for (A.keys_log = 0; (1 << A.keys_log) < A.keys;) ++A.keys_log;
    return true;
}

enum class Family { kGeneral, kWarp, kTc };
struct Chosen { Args A; Family family; bool aligned; int warps; size_t workspace; };

size_t workspace_of(const Args& A)
{
    return A.whole ? 0 : (shared_bytes(A.ctas) + 2 * (size_t)A.ctas * slot_bytes(A.M, A.D) + 255) & ~(size_t)255;
}

int choose(const natten_paged_params_t* p, Chosen& c, const void* q, const void* kc, const void* vc)
{
    if (!p || p->batch < 0 || p->length < 0 || p->heads_q <= 0 || p->heads_kv <= 0 || p->dim <= 0 || p->heads_q % p->heads_kv != 0 ||
        p->pages < 0 || p->page_size <= 0 || p->table_width < 0 || p->kernel < 0 || p->dilation <= 0 ||
        p->dtype < NATTEN_F32 || p->dtype > NATTEN_F64)
        return NATTEN_E_INVALID;
    if (p->dtype == NATTEN_F64 || p->dim > 256 || p->length > kAllOfThePast / 2) return NATTEN_E_UNSUPPORTED;
    Args& A = c.A;
    A = Args{};
    A.q = q; A.kc = kc; A.vc = vc;
    A.table = p->page_table; A.cache_lens = p->cache_lens; A.seq_lens = p->seq_lens; A.table_stride = p->table_stride;
    const int width = p->dtype == NATTEN_F32 ? 4 : 2, n = 16 / width;
    c.aligned = p->dim % n == 0 && ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(kc) | reinterpret_cast<uintptr_t>(vc)) & 15u) == 0;
    for (int i = 0; i < 3; ++i) {
        A.qs[i] = p->q_stride[i]; A.ks[i] = p->k_cache_stride[i]; A.vs[i] = p->v_cache_stride[i];
        c.aligned = c.aligned && A.qs[i] % n == 0 && A.ks[i] % n == 0 && A.vs[i] % n == 0;
    }
    A.B = p->batch; A.L = p->length; A.Hq = p->heads_q; A.Hkv = p->heads_kv; A.G = p->heads_q / p->heads_kv; A.D = p->dim;
    A.pages = p->pages; A.page_size = p->page_size; A.table_width = p->table_width;
    A.K = p->kernel == 0 ? kAllOfThePast : std::min(p->kernel, kAllOfThePast);
    // without a window there is one class
    A.dil = p->kernel == 0 ? 1 : std::min(p->dilation, kAllOfThePast);
    A.by_page = FastDiv((uint32_t)p->page_size);
    A.scale_log2 = (float)(p->scale * 1.4426950408889634);
    if (A.B == 0 || A.L == 0) return NATTEN_OK;
    // The workspace serves every family that the call may take with other pointers and strides.
    const bool simt = (p->flags & NATTEN_FLAG_FORCE_SIMT) != 0;
    Shape shape;
    Args general = A;
    if (!general_shape(p->dtype, general, shape) || !divide(general, shape)) return NATTEN_E_UNSUPPORTED;
    c.family = Family::kGeneral;
    c.workspace = workspace_of(general);
    const bool tc = !simt && tc_shape(p->dtype, A, p->dim % 8 == 0, shape);
    c.warps = 8;
    if (tc || (!simt && warp_shape(p->dtype, A, p->dim % 8 == 0, c.warps, shape))) {
        if (!divide(A, shape)) return NATTEN_E_UNSUPPORTED;
        if (!tc && A.whole && (long long)A.columns * A.Hkv > sm_count()) {      // (measured in paged_warp.cu)
            c.warps = 4;
            warp_shape(p->dtype, A, true, c.warps, shape);
            divide(A, shape);
        }
        c.workspace = std::max(c.workspace, workspace_of(A));
        if (c.aligned) c.family = tc ? Family::kTc : Family::kWarp;
    }
    if ((p->flags & NATTEN_FLAG_FORCE_TC) && c.family != Family::kTc) return NATTEN_E_UNSUPPORTED;
    if (c.family == Family::kGeneral) A = general;
    return NATTEN_OK;
}

} // namespace
} // namespace paged
} // namespace natten

using namespace natten;
using namespace natten::paged;

extern "C" {

size_t natten_paged_workspace_bytes(const natten_paged_params_t* p)
{
    Chosen c;
    if (choose(p, c, nullptr, nullptr, nullptr) != NATTEN_OK || c.A.B == 0 || c.A.L == 0) return 0;
    return c.workspace;
}

int natten_paged_fwd(const natten_paged_params_t* p, const void* q, const void* k_cache, const void* v_cache, void* out, void* lse,
                     void* workspace, size_t workspace_bytes, void* stream)
{
    Chosen c;
    const int rc = choose(p, c, q, k_cache, v_cache);
    if (rc) return rc;
    Args& A = c.A;
    if (A.B == 0 || A.L == 0) return NATTEN_OK;
    if (!q || !out || !A.cache_lens || (A.table_width > 0 && !A.table) || (A.pages > 0 && (!k_cache || !v_cache))) return NATTEN_E_INVALID;
    if (c.workspace > 0 && (workspace_bytes < c.workspace || !workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u))) return NATTEN_E_WORKSPACE;
    A.out = out;
    A.lse = static_cast<float*>(lse);
    A.ws = static_cast<unsigned char*>(workspace);
    const cudaStream_t s = (cudaStream_t)stream;
    note_path(c.family == Family::kTc ? NATTEN_PATH_TCGEN05 : c.family == Family::kWarp ? NATTEN_PATH_WARP : NATTEN_PATH_SIMT);
    const int err = c.family == Family::kTc ? tc_run(p->dtype, A, s) : c.family == Family::kWarp ? warp_run(p->dtype, A, c.warps, s)
                                                                                               : general_run(p->dtype, A, c.aligned, s);
    return err || A.whole ? err : join(p->dtype, A, s);
}

} // extern "C"
