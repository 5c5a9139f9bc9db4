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

namespace natten {
namespace paged {
namespace {

constexpr int kJoinThreads = 128;

template <typename T> __device__ __forceinline__ T rounded(float x);
template <> __device__ __forceinline__ float rounded(float x) { return x; }
template <> __device__ __forceinline__ __half rounded(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 rounded(float x) { return __float2bfloat16_rn(x); }

// Block (c, y): rows y * 4 ... of the unit that CTA c's piece ends inside of, a row a warp.  Its parts are in slot 2c + 1 and in
// slots 2(c + 1), 2(c + 2), ... up to the CTA that finishes the unit.  With M = max m_i: sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i.
template <typename T> __global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ Args A)
{
    const int c = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Shared* all = reinterpret_cast<const Shared*>(A.ws);
    const int unit = all[c].tail;
    if (unit < 0) return;
    const int column = unit / A.Hkv, h = unit - column * A.Hkv;
    const Tile x = tile_of(A, column);
    const int row = blockIdx.y * (kJoinThreads / 32) + warp;
    if (row >= x.rows) return;
    int parts = 1;                           // CTAs of the unit
    for (bool on = true; on;) {
        const int k = c + parts + lane;
        const bool part = k < A.ctas && all[k].head == unit;
        const unsigned ends = __ballot_sync(0xffffffffu, !part || all[k].head_done);
        if (ends) {
            const int e = __ffs(ends) - 1;
            parts += e + (__shfl_sync(0xffffffffu, (int)part, e) ? 1 : 0);
            on = false;
        } else {
            parts += 32;
        }
    }
    auto slot = [&](int i) { return i == 0 ? 2 * c + 1 : 2 * (c + i); };
    float top = -CUDART_INF_F;
    bool bad = false;                        // a NaN maximum
    for (int i = lane; i < parts; i += 32) {
        const float m = slot_sums(A, slot(i))[row].x;
        bad = bad || m != m;
        top = fmaxf(top, m);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (__any_sync(0xffffffffu, bad)) top = CUDART_NAN_F;
    const float base = top == -CUDART_INF_F ? 0.f : top;
    float total = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < parts; ++i) {
        const float2 ml = slot_sums(A, slot(i))[row];
        const float f = exp2f(ml.x - base);
        total = fmaf(f, ml.y, total);
        if (f == 0.f) continue;              // a part that saw nothing
        const float* o = slot_out(A, slot(i)) + (long long)row * A.D;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (lane + 32 * e < A.D) acc[e] = fmaf(f, o[lane + 32 * e], acc[e]);
    }
    long long index;
    int t;
    row_of(A, x, h, row, index, t);
    const float inv = total > 0.f ? 1.f / total : total;
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (lane + 32 * e < A.D) static_cast<T*>(A.out)[index * A.D + lane + 32 * e] = rounded<T>(acc[e] * inv);
    if (A.lse && lane == 0) A.lse[index] = total == 0.f ? -CUDART_INF_F : (base + log2f(total)) * 0.6931471805599453f;
}

int join(int dtype, const Args& A, cudaStream_t s)
{
    const dim3 grid(A.ctas, (A.M + kJoinThreads / 32 - 1) / (kJoinThreads / 32));
    if (dtype == NATTEN_F32) join_kernel<float><<<grid, kJoinThreads, 0, s>>>(A);
    else if (dtype == NATTEN_F16) join_kernel<__half><<<grid, kJoinThreads, 0, s>>>(A);
    else join_kernel<__nv_bfloat16><<<grid, kJoinThreads, 0, s>>>(A);
    simt_count_launch(1);
    return (int)cudaGetLastError();
}

// Tile counts of the padded batch, whatever the lengths are.  False: more units than 31 bits number.
bool divide(Args& A, const Shape& shape)
{
    A.M = shape.M;
    A.keys = shape.keys;
    A.overhead = shape.overhead;
    A.least = shape.least;
    A.align = 1;
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
    return true;
}

enum class Family { kGeneral, kWarp, kTc };
struct Chosen { Args A; Family family; bool aligned; size_t workspace; };

size_t workspace_of(const Args& A) { return (shared_bytes(A.ctas) + 2 * (size_t)A.ctas * slot_bytes(A.M, A.D) + 255) & ~(size_t)255; }

int choose(const natten_paged_params_t* p, Chosen& c, const void* q, const void* kc, const void* vc)
{
    if (!p || p->batch < 0 || p->length < 0 || p->heads_q <= 0 || p->heads_kv <= 0 || p->dim <= 0 || p->heads_q % p->heads_kv != 0 ||
        p->pages < 0 || p->page_size <= 0 || p->table_width < 0 || p->kernel < 0 || p->dilation <= 0 ||
        p->dtype < NATTEN_F32 || p->dtype > NATTEN_F64)
        return NATTEN_E_INVALID;
    if (p->dtype == NATTEN_F64 || p->dim > 256) return NATTEN_E_UNSUPPORTED;
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
    // without a window there is one class, and classes that no two tokens can be in are all alike
    A.dil = p->kernel == 0 ? 1 : p->dilation;
    A.by_page = FastDiv((uint32_t)p->page_size);
    A.scale_log2 = (float)(p->scale * 1.4426950408889634);
    if (A.B == 0 || A.L == 0) return NATTEN_OK;
    // The workspace serves every family that the call may take with other pointers and strides.
    const bool simt = (p->flags & NATTEN_FLAG_FORCE_SIMT) != 0;
    Shape shape;
    Args general = A;
    if (!general_shape(p->dtype, general, c.aligned, shape) || !divide(general, shape)) return NATTEN_E_UNSUPPORTED;
    c.family = Family::kGeneral;
    c.workspace = workspace_of(general);
    const bool tc = !simt && tc_shape(p->dtype, A, p->dim % 8 == 0, shape);
    if (tc || (!simt && warp_shape(p->dtype, A, p->dim % 8 == 0, shape))) {
        if (!divide(A, shape)) return NATTEN_E_UNSUPPORTED;
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
    if (workspace_bytes < c.workspace || !workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u)) return NATTEN_E_WORKSPACE;
    A.out = out;
    A.lse = static_cast<float*>(lse);
    A.ws = static_cast<unsigned char*>(workspace);
    const cudaStream_t s = (cudaStream_t)stream;
    note_path(c.family == Family::kTc ? NATTEN_PATH_TCGEN05 : c.family == Family::kWarp ? NATTEN_PATH_WARP : NATTEN_PATH_SIMT);
    const int err = c.family == Family::kTc ? tc_run(p->dtype, A, s) : c.family == Family::kWarp ? warp_run(p->dtype, A, s)
                                                                                               : general_run(p->dtype, A, c.aligned, s);
    return err ? err : join(p->dtype, A, s);
}

} // extern "C"
