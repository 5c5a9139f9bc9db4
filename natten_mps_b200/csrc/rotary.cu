// Rotary positions of queries and keys, and the append of new keys and values to a paged cache with the rotation applied on
// the way: one kernel, one pass over the data.
//
// A channel pair (a, b) of a token at position p is turned by the angle p * f of its frequency,
//     a' = m (a cos - b sin),   b' = m (b cos + a sin),
// and its gradient by the negative angle.  Angles are the same for every head of a token: a block takes a few tokens, computes
// their cosines and sines once into shared memory (the angle in turns, reduced to [-1/2, 1/2] in 64 bits, so that far positions
// keep their accuracy; the cosine and sine of what is left in 32), and then streams all heads of q, k and v, 16 bytes of each
// half of a pair at a time.
//
// Bound by memory in principle (6 operations a pair against 8 bytes in 16 bits); measured on one B200, 2 x 8191 tokens of 16 + 4 heads
// of 128, bf16: 36 us a direction, 4.7 TB/s of 6.5, with 55 - 60 % of the issue slots taken.  One token
// for each of 64 sequences: 3.5 us in a graph.  Other shapes of it were slower: a thread that keeps a channel's angles and walks the heads 53 us a direction, four units under way a thread 70, rows across threadIdx.y 37.
#include "../../include/natten_b200.h"

#include "device_cache.cuh"
#include "fast_div.cuh"
#include "simt_kernels.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstring>
#include <type_traits>

namespace natten {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 16;              // tokens a block takes at most

struct TurnArgs {
    const void *q, *k, *v;
    void *q_out, *k_out, *v_out;            // k_out, v_out: the caches when there is a page table
    const double* freq;
    const int64_t* positions;
    const int *table, *cache_lens, *seq_lens;
    int64_t pos_stride[2], qs[3], ks[3], vs[3];
    int64_t kd[3], vd[3], table_stride;     // k_out / v_out: page (or batch), token, head
    long long tokens;                       // batch * length
    int length, hq, hk, hv, dim, half;      // half: rotated pairs of a head
    int pages, page_size, table_width, per_block;
    int pair_units, row_units, copy_units;  // units of a rotated row that turn, in all; units of a row of v
    FastDiv by_length, by_token, by_row, by_copy, by_page;
    double magnitude;
    int inverse;
};

struct Token {
    long long k_dst, v_dst, in;             // destinations (elements), index in the padded batch (-1: none)
    int b, i;
    bool live, kept;                        // a new token of its sequence; its slot in the cache is there
};

template <typename T> struct Acc { using type = float; };
template <> struct Acc<double> { using type = double; };

__device__ __forceinline__ float up(float x) { return x; }
__device__ __forceinline__ float up(__half x) { return __half2float(x); }
__device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ double up(double x) { return x; }
template <typename T, typename A> __device__ __forceinline__ T down(A x)
{
    if constexpr (std::is_same<T, __half>::value) return __float2half_rn(x);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __float2bfloat16_rn(x);
    else return x;
}

__device__ __forceinline__ void sin_cos_pi(float x, float& s, float& c) { sincospif(x, &s, &c); }
__device__ __forceinline__ void sin_cos_pi(double x, double& s, double& c) { sincospi(x, &s, &c); }

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Vec { T x[VEC]; };

// Nothing that is read is written by the kernel.
template <typename V> __device__ __forceinline__ V fetch(const void* p)
{
    V v;
    if constexpr (sizeof(V) == 16) {
        const uint4 x = __ldg(static_cast<const uint4*>(p));
        memcpy(&v, &x, 16);
    } else {
        v = *static_cast<const V*>(p);
    }
    return v;
}

// position of token `n` of the padded batch, and whether its sequence has it
__device__ __forceinline__ long long position_of(const TurnArgs& A, long long n, int& b, int& i, bool& live)
{
    b = A.by_length.div(static_cast<int>(n));
    i = static_cast<int>(n) - b * A.length;
    if (!A.table) {
        live = true;
        return A.positions ? A.positions[b * A.pos_stride[0] + i * A.pos_stride[1]] : i;
    }
    const int fresh = A.seq_lens ? min(max(A.seq_lens[b], 0), A.length) : A.length;
    live = i < fresh;
    return static_cast<long long>(A.cache_lens[b]) - fresh + i;
}

template <typename T, int VEC, bool INTER>
__global__ void __launch_bounds__(kThreads) turn_kernel(const __grid_constant__ TurnArgs A)
{
    using acc = typename Acc<T>::type;
    using V = Vec<T, VEC>;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    __shared__ Token toks[kMaxTokens];
    acc* cosv = reinterpret_cast<acc*>(smem_raw);           // [per_block][half]
    acc* sinv = cosv + A.per_block * A.half;
    const int tid = threadIdx.x;
    const long long first = static_cast<long long>(blockIdx.x) * A.per_block;

    for (int e = tid; e < A.per_block * A.half; e += kThreads) {
        const int t = e / A.half, j = e - t * A.half;
        if (first + t >= A.tokens) break;
        int b, i;
        bool live;
        const long long pos = position_of(A, first + t, b, i, live);
        const double turns = static_cast<double>(pos) * (A.freq[j] * 0.15915494309189533577);      // 1 / (2 pi)
        acc s, c;
        sin_cos_pi(static_cast<acc>(2.0 * (turns - rint(turns))), s, c);
        const acc m = static_cast<acc>(A.magnitude);
        cosv[e] = c * m;
        sinv[e] = (A.inverse ? -s : s) * m;
    }
    if (tid < A.per_block) {
        Token k;
        k.in = first + tid < A.tokens ? first + tid : -1;
        k.live = k.kept = false;
        k.k_dst = k.v_dst = 0;
        k.b = k.i = 0;
        if (k.in >= 0) {
            const long long pos = position_of(A, k.in, k.b, k.i, k.live);
            if (A.table) {
                const int p = static_cast<int>(pos);
                const int n = pos >= 0 && pos < 0x7fffffffll ? A.by_page.div(p) : A.table_width;
                if (k.live && pos >= 0 && n < A.table_width) {
                    const int page = A.table[k.b * A.table_stride + n], off = p - n * A.page_size;
                    k.kept = page >= 0 && page < A.pages;
                    k.k_dst = page * A.kd[0] + off * A.kd[1];
                    k.v_dst = page * A.vd[0] + off * A.vd[1];
                }
            } else {
                k.kept = true;
                k.k_dst = k.b * A.kd[0] + k.i * A.kd[1];
            }
        }
        toks[tid] = k;
    }
    __syncthreads();

    const int rotated = (A.hq + A.hk) * A.row_units, all = rotated + A.hv * A.copy_units;
    for (int e = tid; e < A.per_block * all; e += kThreads) {
        const int t = A.by_token.div(e);
        const Token& k = toks[t];
        if (k.in < 0) break;                               // tokens run out: so they do for every later unit
        int w = e - t * all;
        const T* src;
        T* dst;
        int a, b = -1;                                     // channels of the unit's vectors; b < 0: one vector
        bool turned = false;
        bool zero = false;
        if (w < rotated) {
            int h = A.by_row.div(w);
            const int u = w - h * A.row_units;
            if (u < A.pair_units) {
                turned = true;
                a = (INTER && VEC == 1 ? 2 : 1) * u * VEC;
                b = INTER ? (VEC == 1 ? a + 1 : -1) : a + A.half;
            } else {
                a = 2 * A.half + (u - A.pair_units) * VEC;
            }
            if (h < A.hq) {
                src = static_cast<const T*>(A.q) + k.b * A.qs[0] + k.i * A.qs[1] + h * A.qs[2];
                dst = static_cast<T*>(A.q_out) + (k.in * A.hq + h) * A.dim;
                zero = !k.live;
            } else {
                if (!k.kept) continue;
                h -= A.hq;
                src = static_cast<const T*>(A.k) + k.b * A.ks[0] + k.i * A.ks[1] + h * A.ks[2];
                dst = static_cast<T*>(A.k_out) + k.k_dst + h * A.kd[2];
            }
        } else {
            if (!k.kept) continue;
            w -= rotated;
            const int h = A.by_copy.div(w);
            a = (w - h * A.copy_units) * VEC;
            src = static_cast<const T*>(A.v) + k.b * A.vs[0] + k.i * A.vs[1] + h * A.vs[2];
            dst = static_cast<T*>(A.v_out) + k.v_dst + h * A.vd[2];
        }
        V x, y;
        if (zero) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) x.x[i] = y.x[i] = down<T>(acc(0));
        } else {
            x = fetch<V>(src + a);
            if (b >= 0) y = fetch<V>(src + b);
            if (turned) {
                if constexpr (INTER && VEC > 1) {
                    const acc *cs = cosv + t * A.half + a / 2, *sn = sinv + t * A.half + a / 2;
#pragma unroll
                    for (int i = 0; i < VEC / 2; ++i) {
                        const acc p = up(x.x[2 * i]), r = up(x.x[2 * i + 1]), c = cs[i], s = sn[i];
                        x.x[2 * i] = down<T>(p * c - r * s);
                        x.x[2 * i + 1] = down<T>(r * c + p * s);
                    }
                } else {
                    const int j = INTER ? a / 2 : a;
                    const acc *cs = cosv + t * A.half + j, *sn = sinv + t * A.half + j;
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        const acc p = up(x.x[i]), r = up(y.x[i]), c = cs[i], s = sn[i];
                        x.x[i] = down<T>(p * c - r * s);
                        y.x[i] = down<T>(r * c + p * s);
                    }
                }
            }
        }
        *reinterpret_cast<V*>(dst + a) = x;
        if (b >= 0) *reinterpret_cast<V*>(dst + b) = y;
    }
}

size_t width_of(int dtype) { return dtype == NATTEN_F64 ? 8 : dtype == NATTEN_F32 ? 4 : 2; }

// 16-byte vectors: every row of every tensor starts on a 16-byte boundary, and neither half of a pair is cut.
bool vectors_fit(const TurnArgs& A, int dtype, bool interleaved)
{
    const int64_t n = 16 / (int64_t)width_of(dtype);
    bool ok = A.dim % n == 0 && 2 * A.half % n == 0 && (interleaved || A.half % n == 0);
    for (const void* p : {A.q, A.k, A.v, (const void*)A.q_out, (const void*)A.k_out, (const void*)A.v_out})
        ok = ok && (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
    for (int i = 0; i < 3; ++i)
        ok = ok && (!A.q || A.qs[i] % n == 0) && (!A.k || (A.ks[i] % n == 0 && A.kd[i] % n == 0)) &&
             (!A.v || (A.vs[i] % n == 0 && A.vd[i] % n == 0));
    return ok;
}

int launch_turn(TurnArgs& A, int dtype, bool interleaved, cudaStream_t stream)
{
    if (A.tokens == 0) return NATTEN_OK;
    if (A.tokens > 0x7fffffffll - kMaxTokens) return NATTEN_E_UNSUPPORTED;
    const bool vec = vectors_fit(A, dtype, interleaved);
    const int n = vec ? 16 / (int)width_of(dtype) : 1;
    A.pair_units = vec && interleaved ? 2 * A.half / n : A.half / n;
    A.row_units = A.pair_units + (A.dim - 2 * A.half) / n;
    A.copy_units = A.dim / n;
    const int per_token = (A.hq + A.hk) * A.row_units + A.hv * A.copy_units;
    // About four units a thread, as long as every SM still gets blocks enough to hide its latencies.
    long long t = std::max(1, 4 * kThreads / per_token);
    t = std::min<long long>(t, std::max<long long>(1, A.tokens / (4 * sm_count())));
    const size_t acc = dtype == NATTEN_F64 ? 8 : 4;
    t = std::min<long long>({t, kMaxTokens, std::max<long long>(1, (32 << 10) / (long long)(2 * acc * std::max(1, A.half)))});
    A.per_block = (int)t;
    const size_t smem = 2 * acc * (size_t)A.per_block * A.half;
    A.by_length = FastDiv((uint32_t)A.length);
    A.by_token = FastDiv(per_token);
    A.by_row = FastDiv(A.row_units);
    A.by_copy = FastDiv(std::max(1, A.copy_units));
    const long long blocks = (A.tokens + t - 1) / t;
    auto go = [&](auto type, auto width, auto inter) {
        using T = decltype(type);
        turn_kernel<T, decltype(width)::value, decltype(inter)::value><<<(unsigned)blocks, kThreads, smem, stream>>>(A);
    };
    auto by_layout = [&](auto type, auto width) {
        if (interleaved) go(type, width, std::true_type{});
        else go(type, width, std::false_type{});
    };
    auto by_width = [&](auto type) {
        if (vec) by_layout(type, std::integral_constant<int, 16 / (int)sizeof(type)>{});
        else by_layout(type, std::integral_constant<int, 1>{});
    };
    switch (dtype) {
        case NATTEN_F32: by_width(float{}); break;
        case NATTEN_F16: by_width(__half{}); break;
        case NATTEN_BF16: by_width(__nv_bfloat16{}); break;
        default: by_width(double{}); break;
    }
    simt_count_launch(1);
    const cudaError_t err = cudaGetLastError();
    return err == cudaSuccess ? NATTEN_OK : (int)err;
}

// dim <= 1024: a block's table of cosines and sines and its indices stay small
bool sizes_ok(int dtype, int batch, int length, int hq, int hk, int dim, int rotary)
{
    return dtype >= NATTEN_F32 && dtype <= NATTEN_F64 && batch >= 0 && length >= 0 && hq > 0 && hk >= 0 && dim > 0 && rotary >= 0 &&
           rotary <= dim && rotary % 2 == 0;
}
bool sizes_covered(int hq, int hk, int dim) { return dim <= 1024 && (long long)(hq + 2 * hk) * dim <= (1 << 24); }

} // namespace
} // namespace natten

using namespace natten;

extern "C" {

int natten_rotary(const natten_rotary_params_t* p, const void* q, const void* k, void* q_out, void* k_out, void* stream)
{
    if (!p || !sizes_ok(p->dtype, p->batch, p->length, p->heads_q, p->heads_kv, p->dim, p->rotary_dim)) return NATTEN_E_INVALID;
    if (!sizes_covered(p->heads_q, p->heads_kv, p->dim)) return NATTEN_E_UNSUPPORTED;
    TurnArgs A{};
    A.tokens = (long long)p->batch * p->length;
    if (A.tokens == 0) return NATTEN_OK;
    if (A.tokens > 0x7fffffffll - kMaxTokens) return NATTEN_E_UNSUPPORTED;
    if (!q || !q_out || (k == nullptr) != (k_out == nullptr) || (p->rotary_dim > 0 && !p->frequencies)) return NATTEN_E_INVALID;
    A.q = q; A.k = k; A.q_out = q_out; A.k_out = k_out;
    A.freq = p->frequencies;
    A.positions = p->positions;
    for (int i = 0; i < 2; ++i) A.pos_stride[i] = p->position_stride[i];
    for (int i = 0; i < 3; ++i) { A.qs[i] = p->q_stride[i]; A.ks[i] = p->k_stride[i]; }
    A.length = p->length; A.hq = p->heads_q; A.hk = k ? p->heads_kv : 0; A.hv = 0; A.dim = p->dim; A.half = p->rotary_dim / 2;
    A.kd[0] = (int64_t)p->length * p->heads_kv * p->dim; A.kd[1] = (int64_t)p->heads_kv * p->dim; A.kd[2] = p->dim;
    A.magnitude = p->magnitude;
    A.inverse = p->inverse != 0;
    return launch_turn(A, p->dtype, p->interleaved != 0, (cudaStream_t)stream);
}

int natten_paged_append(const natten_paged_params_t* p, const void* q, const void* k, const void* v, void* q_out, void* k_cache,
                        void* v_cache, void* stream)
{
    if (!p || !sizes_ok(p->dtype, p->batch, p->length, p->heads_q, p->heads_kv, p->dim, p->rotary_dim) || p->heads_kv <= 0 ||
        p->pages < 0 || p->page_size <= 0 || p->table_width < 0)
        return NATTEN_E_INVALID;
    if (!sizes_covered(p->heads_q, p->heads_kv, p->dim)) return NATTEN_E_UNSUPPORTED;
    TurnArgs A{};
    A.tokens = (long long)p->batch * p->length;
    if (A.tokens == 0) return NATTEN_OK;
    if (A.tokens > 0x7fffffffll - kMaxTokens) return NATTEN_E_UNSUPPORTED;
    if (!k || !v || (p->pages > 0 && (!k_cache || !v_cache)) || (q == nullptr) != (q_out == nullptr) ||
        (p->table_width > 0 && !p->page_table) || !p->cache_lens || (p->rotary_dim > 0 && !p->frequencies))
        return NATTEN_E_INVALID;
    A.q = q; A.k = k; A.v = v; A.q_out = q_out; A.k_out = k_cache; A.v_out = v_cache;
    A.freq = p->frequencies;
    // A table without entries is not read, but tells the append from the rotation alone.
    A.table = p->table_width > 0 ? p->page_table : p->cache_lens;
    A.cache_lens = p->cache_lens; A.seq_lens = p->seq_lens; A.table_stride = p->table_stride;
    for (int i = 0; i < 3; ++i) {
        A.qs[i] = p->q_stride[i]; A.ks[i] = p->k_stride[i]; A.vs[i] = p->v_stride[i];
        A.kd[i] = p->k_cache_stride[i]; A.vd[i] = p->v_cache_stride[i];
    }
    A.length = p->length; A.hq = q ? p->heads_q : 0; A.hk = A.hv = p->heads_kv; A.dim = p->dim; A.half = p->rotary_dim / 2;
    A.pages = p->pages; A.page_size = p->page_size; A.table_width = p->table_width;
    A.by_page = FastDiv((uint32_t)p->page_size);
    A.magnitude = p->magnitude;
    return launch_turn(A, p->dtype, p->interleaved != 0, (cudaStream_t)stream);
}

} // extern "C"
