// Attention over a paged cache for many rows a unit (chunks of a prompt, whole prompts), 16-bit types, head dims 64 and 128, on
// tcgen05 tensor cores: one persistent CTA per SM, 128-key tiles.
//
//   S = Q K^T                     tcgen05.mma, 128 x 128, Q and K in shared memory, S in TMEM
//   P = 2^(S scale log2(e) - m)   one thread a row, 32 columns at a time, written back as 16 bits over the scores they came from
//   O += P V                      tcgen05.mma with A = P from TMEM, V read MN-major, O in TMEM
//
// Two row halves of 128 rows keep the tensor cores and the exponentials busy at the same time: while the threads of one half turn
// its S into P, the products of the other run.  With more than 128 rows in a class the halves are rows 0 - 127 and 128 - 255 of
// the unit and share every tile of keys; with fewer they take the same rows and every other tile of keys (kSplit), each with its
// own maximum and sum, and are joined at the end.
//
// A row's maximum m is fixed at the first columns that it sees and moves only if a later score exceeds it by 2^60 (float16: 2^14),
// which the row sum of a piece tells; O, the sum and the tile's probabilities so far are then rescaled by the thread itself.  So
// there is no running maximum, and no thread has to touch O in between.  S scale log2(e) - m is one fused operation, so that a
// score of m's size leaves the rounding of m, half a step, as an exponent: rows with |m| from 2^24 on, where that passes 1/2, take
// the rescaling's own arithmetic, which rounds the product first, as m was.
//
// Sixteen warps: two warpgroups of softmax, one that loads, one warp that issues the products, one that walks the CTA's units and
// hands them to the others (what a unit is takes some hundred instructions and the sequence's lengths, which would stand in
// front of every unit in every role; and the less code the roles have, the less of it is fetched again for every unit).  The loading threads look the keys
// of a tile up in the page table, a tile ahead.  Where 16 or more keys at a time are adjacent in a page (no dilation, a page
// size that is a multiple of 16) tiles start at such a run, and TMA brings the runs that are there as a whole.  The other keys
// (of runs that a unit's first and last key cut, pages of other sizes, dilated keys) are copied row by row, 16 bytes at a time,
// into the same swizzled layout; a row that is not there is zero, whatever its slot holds.  Row-wise copies of every tile would
// take 3750 cycles a tile, twice what the products need.  The queries come by TMA where a group's heads divide the tile, too.
//
// P is rounded to the tensors' type, since the product takes one type: half a step of each weight, where the output itself is rounded
// by as much.  The row sum adds the weights as they were.  Against 64 bits the outputs are off by 0.0022 - 0.0024 of their size in
// bfloat16 and 0.00027 in float16, where the output's rounding alone leaves 0.0017 and 0.00021; a second product with what the
// rounding cut off would bring that back for half as many tensor products again.
//
// Measured on one B200, bf16, 16 heads of 128 on 4: chunks of 2048 tokens over caches of 16384, batch 2, 455 - 464 us at 1.97 GHz
// with pauses (1110 - 1130 TFLOP/s), 519 - 528 us back to back (980 - 990), where the power cap holds the clock at 1.6 GHz; prompts of
// 8191 through a window of 255, batch 2, 91 - 93 us.  The tensor products of a tile are 2048 cycles for both halves, the exponentials 1024 a half on the special-
// function unit; with time stamps in the kernel a tile took 3600 cycles, in which a half spent about 1600 on its exponentials and
// waited about 1100 for its products, behind the other half's.  Short units of a window have masked tiles and outputs instead.
//
// TMEM columns: S (P over its first half) of the halves at 0 and 128, O at 256 and 384.
#include "../../include/natten_b200.h"

#include "device_cache.cuh"
#include "paged.cuh"
#include "tc_common.cuh"
#include "tc_kernels.cuh"
#include "tc_plan.cuh"

#include <math_constants.h>

#include <type_traits>

namespace natten {
namespace paged {

using namespace tc;
using tcplan::add2;
using tcplan::cvt_pack;
using tcplan::fast_exp2;
using tcplan::fma2;
using tcplan::hi_of;
using tcplan::lo_of;
using tcplan::low_bits;
using tcplan::pack2;
using tcplan::transpose4;

namespace {

constexpr int kThreads = 512, kKeys = 128, kHalfRows = 128, kWordSlots = 16, kUnitSlots = 4;
constexpr int kSoftmaxRegs = 176, kHelperRegs = 80;              // 2 x 128 x (176 + 80) = the 65536 of the launch
constexpr uint32_t kColO = 256;

// A unit, or a CTA's part of one: key tiles [x0, x1) of a row tile and a key/value head.
enum : int { kEnd, kWork, kClear };          // kClear: no row sees anything
struct Unit {
    int kind, h, x0, x1, direct;             // direct: rows are written out; else to the CTA's slot of partial results
    Tile tile;
};

struct Status { int* status; int* status_host; long long wait_budget; int inject, boxed; };      // boxed: queries come by TMA

template <int DH, bool SPLIT> struct Cfg {
    static constexpr int kBlocks = DH / 64;                      // 64-channel blocks: rows of 128 bytes, 128-byte swizzle
    static constexpr int kRows = SPLIT ? kHalfRows : 2 * kHalfRows;
    static constexpr int kQBlock = kRows * 128, kBlock = kKeys * 128;
    static constexpr int kQ = kQBlock * kBlocks, kTile = kBlock * kBlocks;
    static constexpr int kStages = DH == 128 ? (SPLIT ? 5 : 4) : 8;
    static constexpr int kOffKV = kQ;
    static constexpr int kOffRows = kOffKV + kStages * kTile;    // long long [3][2][kKeys]: places of a tile's keys and values
    static constexpr int kOffWords = kOffRows + 3 * 2 * kKeys * 8;   // uint4 [kWordSlots]: which keys of a tile are there
    static constexpr int kOffCopied = kOffWords + kWordSlots * 16;   // unsigned [kWordSlots]: were rows of the tile copied?
    static constexpr int kOffSums = kOffCopied + kWordSlots * 4; // float2 [kHalfRows]: the second half's sums (kSplit)
    static constexpr int kOffBars = kOffSums + kHalfRows * 8;
    static constexpr int kBars = 2 * kStages + kWordSlots + 2 + 2 + 2 + 2 + 2 + 2 + 2 * kUnitSlots;
    static constexpr int kOffFlags = kOffBars + 8 * kBars;       // abort flag, TMEM address
    static constexpr int kOffScratch = (kOffFlags + 8 + 15) & ~15;
    static constexpr int kOffUnits = (kOffScratch + (int)sizeof(Piece::Scratch) + 15) & ~15;      // Unit [kUnitSlots]
    static constexpr int kSmem = kOffUnits + kUnitSlots * (int)sizeof(Unit);
    static_assert(kTile % 1024 == 0 && kSmem <= kMaxDynamicSmem, "shared memory of a CTA");
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there)
{
    const int n = there ? 16 : 0;            // 0: nothing is read, the chunk is zero
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void copies_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// The barrier gets this thread's arrival once all copies that it has issued so far have landed.  They are ordinary writes: who reads
// them through the tensor cores puts a proxy fence behind its wait.
__device__ __forceinline__ void arrive_when_landed(uint32_t b)
{
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(b) : "memory");
}
// 2^x of two values on the FMA pipe, for a share of the exponentials (the special-function unit does 16 a cycle, the products of a
// tile leave it one cycle for each): x = n + f with n the nearest whole number, 2^f by the polynomial of degree 4 with the least
// largest relative error on [-1/2, 1/2] (2.6e-6, from a Remez exchange), n added to the exponent.  Values above 127 and NaN give 2^127,
// which the tile's sum tells.
__device__ __forceinline__ void exp2_fma(uint64_t e, float& a, float& b)
{
    const uint64_t x = pack2(fmaxf(fminf(lo_of(e), 127.f), -126.f), fmaxf(fminf(hi_of(e), 127.f), -126.f));
    constexpr float kRound = 12582912.f;     // 1.5 * 2^23: adding it leaves the nearest whole number in the low bits
    const uint64_t r = add2(x, pack2(kRound, kRound)), n = add2(r, pack2(-kRound, -kRound)), f = fma2(n, pack2(-1.f, -1.f), x);
    uint64_t y = fma2(pack2(0.009570102207362652f, 0.009570102207362652f), f, pack2(0.05591785907745361f, 0.05591785907745361f));
    y = fma2(y, f, pack2(0.240247443318367f, 0.240247443318367f));
    y = fma2(y, f, pack2(0.6931217908859253f, 0.6931217908859253f));
    y = fma2(y, f, pack2(0.9999992847442627f, 0.9999992847442627f));
    a = __uint_as_float(__float_as_uint(lo_of(y)) + (__float_as_uint(lo_of(r)) << 23));
    b = __uint_as_float(__float_as_uint(hi_of(y)) + (__float_as_uint(hi_of(r)) << 23));
}
// The barrier's phase waits for these bytes, too (no arrival).
__device__ __forceinline__ void mbar_expect_bytes(uint32_t bar, uint32_t bytes)
{
    asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// The loads of this thread's TMEM rows have landed.  What is done with them takes the returned factor, so that none of it can move
// in front of the wait.  (The loaded registers as operands of the wait would say the same, and measured the same.)
__device__ __forceinline__ uint64_t landed(uint64_t factor)
{
    asm volatile("tcgen05.wait::ld.sync.aligned;" : "+l"(factor) :: "memory");
    return factor;
}
__device__ __forceinline__ float landed(float factor)
{
    asm volatile("tcgen05.wait::ld.sync.aligned;" : "+f"(factor) :: "memory");
    return factor;
}
// barrier 1 of the 128 loading threads; true if every one of them brought true
__device__ __forceinline__ bool loaders_agree(bool ok)
{
    int all;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbarrier.cta.red.and.pred q, 1, 128, p;\n\tselp.b32 %0, 1, 0, q;\n\t}"
                 : "=r"(all) : "r"((int)ok) : "memory");
    return all != 0;
}

template <int DH, bool BF16, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1) tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
          const __grid_constant__ Args A,
          const __grid_constant__ Status P)
{
    using C = Cfg<DH, SPLIT>;
    constexpr int ST = C::kStages;
    extern __shared__ __align__(1024) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t sbase = smem_u32(smem);
    const int prior_abort = *reinterpret_cast<volatile int*>(P.status);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::kOffFlags);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kOffFlags + 4);
    uint32_t bar = sbase + C::kOffBars;
    const uint32_t bar_full = bar;                               // [ST] a tile of keys or values has landed
    const uint32_t bar_empty = bar_full + 8 * ST;                // [ST] ... its products are done
    const uint32_t bar_words = bar_empty + 8 * ST;               // [kWordSlots] which keys of the tile are there
    const uint32_t bar_q = bar_words + 8 * kWordSlots;           // Q of the unit has landed
    const uint32_t bar_qfree = bar_q + 8;                        // the unit's last S is done
    const uint32_t bar_s = bar_qfree + 8;                        // [2] S of the half's tile is in TMEM, and every earlier product is done
    const uint32_t bar_p = bar_s + 16;                           // [2] every thread of the half stored its P
    const uint32_t bar_o = bar_p + 16;                           // [2] the half's last P V of the unit is done
    const uint32_t bar_ofree = bar_o + 16;                       // [2] O has been read
    const uint32_t bar_sums = bar_ofree + 16;                    // [2] kSplit: the second half's sums are in shared memory; have been read

    const uint32_t bar_unit = bar_sums + 16;                     // [kUnitSlots] the unit is there
    const uint32_t bar_unitfree = bar_unit + 8 * kUnitSlots;     // [kUnitSlots] ... has been read by the 13 warps that use it

    if (warp == 12) {
        if (lane == 0) {
            // swizzled tiles need a 1024-byte aligned base; once any CTA has given up, the rest bail out
            *abort_flag = ((sbase & 1023u) || prior_abort) ? 1 : 0;
            for (int i = 0; i < ST; ++i) {
                mbar_init(bar_full + 8 * i, 128);
                mbar_init(bar_empty + 8 * i, 1);
            }
            for (int i = 0; i < kWordSlots; ++i) mbar_init(bar_words + 8 * i, 4);
            for (int i = 0; i < kUnitSlots; ++i) {
                mbar_init(bar_unit + 8 * i, 1);
                mbar_init(bar_unitfree + 8 * i, 13);
            }
            mbar_init(bar_q, 128);
            mbar_init(bar_qfree, 1);
            for (int i = 0; i < 2; ++i) {
                mbar_init(bar_s + 8 * i, 1);
                mbar_init(bar_p + 8 * i, 128);
                mbar_init(bar_o + 8 * i, 1);
                mbar_init(bar_ofree + 8 * i, 128);
                mbar_init(bar_sums + 8 * i, 128);
            }
            mbar_init_fence();
            fence_async_smem();
        }
        __syncwarp();
        tmem_alloc(smem_u32(tmem_slot), 512);
    }
    Piece piece;
    piece.begin<kThreads>(A, blockIdx.x, reinterpret_cast<Piece::Scratch*>(smem + C::kOffScratch));
    let_dependents_launch();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const Unit* units_at = reinterpret_cast<const Unit*>(smem + C::kOffUnits);
    // The CTA's next unit (kEnd after the last one, or when some wait ran out), for a warp.
    auto next_unit = [&](unsigned& walked) {
        const unsigned slot = walked % kUnitSlots;
        Unit u;
        u.kind = kEnd;
        if (warp_wait(bar_unit + 8 * slot, (walked / kUnitSlots) & 1, abort_flag, P.wait_budget)) {
            u = units_at[slot];
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_unitfree + 8 * slot);
        }
        ++walked;
        return u;
    };

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kHelperRegs));
        if (warp == 13) {
            // =====================================================================
            // Units
            // =====================================================================
            Shared told{-1, 0};
            for (unsigned walked = 0; !gave_up(abort_flag); ++walked) {
                Piece::Portion p{};
                bool clear = false;
                while (piece.more()) {
                    p = piece.portion(A);
                    clear = piece.tile.n == 0 && p.first;
                    if (p.work || clear) break;
                    piece.advance(A);
                }
                const bool more = piece.more();
                Unit u;
                u.kind = !more ? kEnd : p.work ? kWork : kClear;
                u.h = p.h; u.x0 = p.x0; u.x1 = p.x1;
                u.direct = clear || p.whole;
                u.tile = piece.tile;
                if (more && !u.direct && p.x0 == 0) told = {piece.column * A.Hkv + p.h, piece.parts(A, blockIdx.x)};
                const unsigned slot = walked % kUnitSlots;
                if (walked >= (unsigned)kUnitSlots &&
                    !warp_wait(bar_unitfree + 8 * slot, (walked / kUnitSlots - 1) & 1, abort_flag, P.wait_budget))
                    break;
                if (lane == 0) {
                    reinterpret_cast<Unit*>(smem + C::kOffUnits)[slot] = u;
                    mbar_arrive(bar_unit + 8 * slot);
                }
                __syncwarp();
                if (!more) break;
                piece.advance(A);
            }
            if (lane == 0 && !A.whole) reinterpret_cast<Shared*>(A.ws)[blockIdx.x] = told;
        } else if (warp == 12) {
            // =====================================================================
            // MMA issue: the whole warp walks the units, the instructions execute on one elected lane.
            // =====================================================================
            bool ok = !gave_up(abort_flag);
            constexpr uint32_t idesc_qk = instr_desc(BF16 ? 1 : 0, kKeys, 0, 0), idesc_pv = instr_desc(BF16 ? 1 : 0, DH, 0, 1);
            const uint32_t leader = elect_one();
            unsigned fills = 0, units[2] = {0, 0}, tiles[2] = {0, 0};           // tiles of keys and values taken; units, tiles of each half
            unsigned queries = 0, seq = 0;                       // units; tiles of the CTA
            bool copied = false;                                 // rows of the tile whose keys came last were copied
            for (unsigned walked = 0; ok;) {
                const Unit u = next_unit(walked);
                if (u.kind == kEnd) break;
                if (u.kind != kWork) continue;
                const int n = u.x1 - u.x0;
                const bool two = SPLIT ? n > 1 : u.tile.rows > kHalfRows;
                auto wait_full = [&]() { ok = ok && mbar_wait(bar_full + 8 * (fills % ST), (fills / ST) & 1, abort_flag, P.wait_budget); };
                // The keys of the next tile have landed.  Rows that threads copied are ordinary writes, which the tensor cores see
                // behind a proxy fence (some hundred cycles on the chain of every tile: not for those that TMA brought).
                auto wait_keys = [&]() {
                    const unsigned w = seq % kWordSlots;
                    ok = ok && mbar_wait(bar_words + 8 * w, (seq / kWordSlots) & 1, abort_flag, P.wait_budget);
                    copied = reinterpret_cast<volatile unsigned*>(smem + C::kOffCopied)[w] != 0u;
                    ++seq;
                    wait_full();
                    if (copied) fence_async_smem();
                };
                auto scores = [&](int half) {
                    const uint64_t dq = smem_desc(sbase + (SPLIT ? 0 : half * kHalfRows * 128), 16, 1024),
                                   dk = smem_desc(sbase + C::kOffKV + (fills % ST) * C::kTile, 16, 1024);
#pragma unroll
                    for (int k = 0; k < DH / 16; ++k)            // 32 bytes per step inside a 64-channel block
                        mma_ss_e(tmem + 128 * half, dq + (((k / 4) * C::kQBlock + (k % 4) * 32) >> 4),
                                 dk + (((k / 4) * C::kBlock + (k % 4) * 32) >> 4), idesc_qk, k > 0, leader);
                    mma_commit_e(bar_s + 8 * half, leader);
                };
                auto weighted = [&](int half, bool first) {
                    const uint64_t dv = smem_desc(sbase + C::kOffKV + (fills % ST) * C::kTile, C::kBlock, 1024);
#pragma unroll
                    for (int k = 0; k < kKeys / 16; ++k)         // 16 keys per step: 16 rows of V, 8 columns of P
                        mma_ts_e(tmem + kColO + 128 * half, tmem + 128 * half + 8 * k, dv + 128 * k, idesc_pv, (!first || k > 0) ? 1u : 0u, leader);
                };
                auto release = [&]() {
                    mma_commit_e(bar_empty + 8 * (fills % ST), leader);
                    ++fills;
                };
                auto wait_p = [&](int half, bool first) {
                    if (first && units[half] > 0) ok = ok && mbar_wait(bar_ofree + 8 * half, (units[half] - 1) & 1, abort_flag, P.wait_budget);
                    ok = ok && mbar_wait(bar_p + 8 * half, tiles[half] & 1, abort_flag, P.wait_budget);
                    ++tiles[half];
                };
                ok = ok && mbar_wait(bar_q, queries & 1, abort_flag, P.wait_budget);
                ++queries;
                wait_keys();
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                if (!P.boxed) fence_async_smem();
                tc_fence_after();
                if constexpr (SPLIT) {
                    // tile j belongs to half j & 1; order of the loads: K0, K1, V0, K2, V1, ...
                    scores(0);
                    if (n == 1) mma_commit_e(bar_qfree, leader);
                    release();
                    for (int j = 0; j < n; ++j) {
                        const bool v_copied = copied;            // tile j's; wait_keys has the next one's
                        if (j + 1 < n) {
                            wait_keys();
                            if (!ok) break;
                            tc_fence_after();
                            scores((j + 1) & 1);                 // after P V of tile j - 1 in issue order: over its P
                            if (j + 2 == n) mma_commit_e(bar_qfree, leader);
                            release();
                        }
                        wait_full();
                        if (v_copied) fence_async_smem();
                        wait_p(j & 1, j < 2);
                        if (!ok) break;
                        tc_fence_after();
                        weighted(j & 1, j < 2);
                        release();
                        if (j + 2 >= n) mma_commit_e(bar_o + 8 * (j & 1), leader);
                    }
                } else {
                    // both halves use every tile; order of the loads: K0, V0, K1, V1, ...
                    scores(0);
                    if (two) scores(1);
                    if (n == 1) mma_commit_e(bar_qfree, leader);
                    release();
                    for (int j = 0; j < n; ++j) {
                        // Everything that can be waited for ahead is: what lies between a half's P and its next S is on the chain
                        // of every tile.
                        const unsigned v = fills;                // V of the tile; K of the next one follows it
                        const bool more = j + 1 < n;
                        wait_full();
                        if (copied) fence_async_smem();          // (still tile j's)
                        fills = v + 1;
                        if (more) wait_keys();
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            if (half == 1 && !two) break;
                            wait_p(half, j == 0);
                            if (!ok) break;
                            tc_fence_after();
                            fills = v;
                            weighted(half, j == 0);
                            if (!more) mma_commit_e(bar_o + 8 * half, leader);
                            fills = v + 1;
                            if (more) scores(half);
                        }
                        if (!ok) break;
                        fills = v;
                        release();                               // V
                        if (more) {
                            if (j + 2 == n) mma_commit_e(bar_qfree, leader);
                            release();                           // K of the next tile
                        }
                    }
                }
                ++units[0];
                if (two) ++units[1];
                if (!__all_sync(0xffffffffu, ok)) ok = false;    // the lanes agree once a unit
            }
        } else if (warp < 12) {
            // =====================================================================
            // Loads
            // =====================================================================
            const int lt = tid - 256;
            const uint16_t *q = static_cast<const uint16_t*>(A.q), *kc = static_cast<const uint16_t*>(A.kc), *vc = static_cast<const uint16_t*>(A.vc);
            long long* places = reinterpret_cast<long long*>(smem + C::kOffRows);      // [3][K: kKeys, V: kKeys]
            constexpr int kChunks = DH / 8, kAtOnce = 128 / kChunks;   // 16-byte chunks of a row; rows at a time
            const int c = lt % kChunks, r0 = lt / kChunks;
            const uint32_t c_off = (c >> 3) * C::kBlock, cq_off = (c >> 3) * C::kQBlock;
            bool ok = loaders_agree(!*abort_flag);
            unsigned fills = 0, seq = 0, queries = 0;
            auto wait_empty = [&](uint32_t b, uint32_t parity) { ok = ok && mbar_wait(b, parity, abort_flag, P.wait_budget); };
            // A tile's keys: this thread's (the lt-th) page and slot, and where the keys and values of all of them are (elements).
            // runs: bit i is set where the run of A.align keys that key i * 16 belongs to is there as a whole.
            struct Keys { int page, slot; unsigned runs; const long long* at; };
            for (unsigned walked = 0;;) {
                const Unit p = next_unit(walked);
                if (p.kind == kEnd) ok = false;
                ok = loaders_agree(ok);
                if (!ok) break;
                if (p.kind != kWork) continue;
                const Tile& x = p.tile;
                const int n = p.x1 - p.x0;
                auto fill = [&](const CUtensorMap* map, const uint16_t* src, const Keys& k, int offset) {
                    const unsigned s = fills % ST;
                    const uint32_t full = bar_full + 8 * s, dst = sbase + C::kOffKV + s * C::kTile;
                    if (fills >= (unsigned)ST) wait_empty(bar_empty + 8 * s, (fills / ST - 1) & 1);
                    if (ok) {
                        if (lt == 0 && k.runs) mbar_expect_bytes(full, __popc(k.runs) * (C::kTile / 8));
                        if (((k.runs >> (lt >> 4)) & 1u) && (lt & (A.align - 1)) == 0)
#pragma unroll
                            for (int b = 0; b < C::kBlocks; ++b)
                                tma_load_5d(dst + b * C::kBlock + lt * 128, map, full, 0, k.slot, b, p.h, k.page);
                        if (k.runs == 0xffu) {
                            mbar_arrive(full);
                        } else {
                            for (int r16 = 0; r16 < kKeys; r16 += 16) {
                                if ((k.runs >> (r16 >> 4)) & 1u) continue;
#pragma unroll
                                for (int r = r16 + r0; r < r16 + 16; r += kAtOnce) {
                                    const long long o = k.at[offset + r];
                                    copy16(dst + c_off + r * 128 + (((c ^ r) & 7) << 4), o >= 0 ? src + o + c * 8 : q, o >= 0);
                                }
                            }
                            arrive_when_landed(full);
                        }
                    }
                    ++fills;
                };
                int page = 0, slot = 0;
                bool there = false;
                auto look_up = [&](int j) {
                    const int t = x.base + (p.x0 + j) * kKeys + lt;
                    there = j < n && t >= x.lo && locate(A, x, t, page, slot);
                };
                look_up(0);
                // Tile j (the lookup for the next one is under way while this one is copied).  Three buffers: with kSplit a thread
                // may still copy the values of tile j - 2 when another writes the places of tile j.
                auto keys_of = [&](int j) {
                    long long* at = places + (j % 3) * 2 * kKeys;
                    const unsigned seen = __ballot_sync(0xffffffffu, there), w = seq % kWordSlots;
                    volatile unsigned* words = reinterpret_cast<volatile unsigned*>(smem + C::kOffWords) + 4 * w;
                    if (lane == 0) words[warp & 3] = seen;
                    at[lt] = there ? page * A.ks[0] + slot * A.ks[1] + p.h * A.ks[2] : -1;
                    at[kKeys + lt] = there ? page * A.vs[0] + slot * A.vs[1] + p.h * A.vs[2] : -1;
                    Keys k{page, slot, 0u, at};
                    look_up(j + 1);
                    ok = loaders_agree(ok);
                    if (A.align > 1) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const unsigned word = words[i];
                            unsigned whole = ((word & 0xffffu) == 0xffffu ? 1u : 0u) | (word >> 16 == 0xffffu ? 2u : 0u);
                            if (A.align > 16) whole = whole == 3u ? 3u : 0u;
                            k.runs |= whole << (2 * i);
                        }
                        if (A.align > 32) k.runs = ((k.runs & 0xfu) == 0xfu ? 0xfu : 0u) | ((k.runs & 0xf0u) == 0xf0u ? 0xf0u : 0u);
                    }
                    if (lane == 0) {
                        if (warp == 8) reinterpret_cast<unsigned*>(smem + C::kOffCopied)[w] = k.runs != 0xffu;
                        mbar_arrive(bar_words + 8 * w);
                    }
                    ++seq;
                    return k;
                };
                auto load_queries = [&]() {
                    if (queries > 0) wait_empty(bar_qfree, (queries - 1) & 1);
                    const bool tell = P.inject != 1 || queries > 0 || lt > 0;        // test hook: a barrier that never fills
                    if (ok && P.boxed) {
                        if (lt == 0) {
                            mbar_expect_bytes(bar_q, C::kQ);
#pragma unroll
                            for (int b = 0; b < C::kBlocks; ++b)
                                tma_load_5d(sbase + b * C::kQBlock, &tmQ, bar_q, 0, p.h * A.G, A.by_group.div(x.row0), b, x.b);
                        }
                        if (tell) mbar_arrive(bar_q);
                    } else if (ok) {
#pragma unroll 2
                        for (int r = r0; r < C::kRows; r += kAtOnce) {
                            const bool here = r < x.rows;
                            copy16(sbase + cq_off + r * 128 + (((c ^ r) & 7) << 4), here ? q + query_offset(A, x, p.h, r) + c * 8 : q, here);
                        }
                        if (tell) arrive_when_landed(bar_q);
                    }
                    ++queries;
                };
                // K0, V0, K1, V1, ...; with kSplit K0, K1, V0, K2, V1, ..., so that the keys are ahead of the other half's values
                Keys keys{}, values{};
#pragma unroll 1
                for (int f = 0; f < 2 * n; ++f) {
                    const bool is_key = SPLIT ? f == 0 || (f & 1 && f < 2 * n - 1) : !(f & 1);
                    const int j = is_key ? (f + 1) / 2 : 0;
                    if (is_key) {
                        const Keys k = keys_of(j);
                        if (!ok) break;
                        values = SPLIT ? keys : k;
                        if (SPLIT && n == 1) values = k;
                        keys = k;
                    } else if (SPLIT && f == 2 * n - 1) {
                        values = keys;
                    }
                    fill(is_key ? &tmK : &tmV, is_key ? kc : vc, is_key ? keys : values, is_key ? 0 : kKeys);
                    if (f == 0) load_queries();
                }
                ok = loaders_agree(ok);                          // the places have been read by everyone
            }
            copies_wait_all();
        }
    } else {
        // =====================================================================
        // Softmax and output: a thread a row
        // =====================================================================
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        constexpr float kGrow = BF16 ? 60.f : 14.f;              // headroom of the stored probabilities, as an exponent
        constexpr float kFar = 16777216.f;                       // 2^24
        constexpr float kGrowSum = BF16 ? 1.152921504606847e18f : 16384.f;     // 2^kGrow: a piece's sum below it has none above it
        const int half = warp >> 2, row = (SPLIT ? 0 : half * kHalfRows) + (warp & 3) * 32 + lane;
        const uint32_t trow = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16), scol = trow + 128 * half, ocol = trow + kColO + 128 * half;
        float2* sums = reinterpret_cast<float2*>(smem + C::kOffSums);
        bool ok = !gave_up(abort_flag);
        unsigned mine = 0, seq = 0, units = 0, exchanges = 0;    // tiles of this half, tiles of the CTA, units of this half
        bool skipped = false;                                    // the last unit, without a look at its tiles
        const uint64_t sc2 = pack2(A.scale_log2, A.scale_log2);
        for (unsigned walked = 0; ok;) {
            const Unit p = next_unit(walked);
            if (p.kind == kEnd) break;
            const Tile& x = p.tile;
            const int n = p.kind == kWork ? p.x1 - p.x0 : 0;
            const bool direct = p.direct;
            const int where = 2 * (int)blockIdx.x + (p.x0 == 0 ? 1 : 0);
            const bool active = SPLIT ? half == 0 || n > 1 : half == 0 || x.rows > kHalfRows;
            if (!active) {
                seq += n;
                skipped = true;
                continue;
            }
            long long index = -1;
            int tq = -1;
            const bool in_tile = row < x.rows;
            bool live = in_tile && row_of(A, x, p.h, row, index, tq);
            if (!in_tile) index = -1;
            const int t_least = __reduce_min_sync(0xffffffffu, live ? tq : 0x7fffffff), t_most = __reduce_max_sync(0xffffffffu, live ? tq : -1);
            if (!live) tq = -1;
            float m = tq >= 0 ? -CUDART_INF_F : 0.f, l = 0.f;    // (rows that do not count hold no tile up)
            float limit = kGrowSum;                              // of a piece's sum; rows far from zero always go past it
            // rare: a score far above the maximum.  Move it; rescale O (its products so far are done, see bar_s), the sum and the
            // probabilities of this tile's first `pieces` pieces.
            auto rescale = [&](bool grow, float to, bool had_tiles, int pieces) {
                const float f = grow ? fast_exp2(m - to) : 1.f;
                tmem_st_wait();
                if (had_tiles) {
#pragma unroll 1
                    for (int part = 0; part < DH / 16; ++part) {
                        uint32_t o[16];
                        tmem_ld16(ocol + 16 * part, o);
                        const float by = landed(f);
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * by);
                        tmem_st16(ocol + 16 * part, o);
                    }
                }
#pragma unroll 1
                for (int pc = 0; pc < pieces; ++pc) {
                    uint32_t w[16];
                    tmem_ld16(scol + 16 * pc, w);
                    const float by = landed(f);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float a, b;
                        if (BF16) {
                            a = __uint_as_float(w[i] << 16);
                            b = __uint_as_float(w[i] & 0xffff0000u);
                        } else {
                            const __half2 h2 = *reinterpret_cast<const __half2*>(&w[i]);
                            a = __low2float(h2);
                            b = __high2float(h2);
                        }
                        w[i] = cvt_pack<BF16>(a * by, b * by);
                    }
                    tmem_st16(scol + 16 * pc, w);
                }
                l *= f;
                if (grow) {
                    m = to;                                      // (m + (to - m) would round to the larger one's step)
                    limit = fabsf(to) < kFar ? kGrowSum : -1.f;
                }
            };
            bool had_tiles = false;
            for (int j = 0; j < n; ++j, ++seq) {
                if (SPLIT && (j & 1) != half) continue;
                const int base = x.base + (p.x0 + j) * kKeys;
                const unsigned w = seq % kWordSlots;
                // A half that left units out may be here long before this tile's words are: their barrier could be two phases
                // behind, which one bit of phase cannot tell from done.  So it waits for the tile's scores first, which are issued
                // behind the words.  With the tile before seen, the words of tile seq - 16 are known to be past.
                if (skipped) ok = ok && mbar_wait(bar_s + 8 * half, mine & 1, abort_flag, P.wait_budget);
                skipped = false;
                ok = ok && mbar_wait(bar_words + 8 * w, (seq / kWordSlots) & 1, abort_flag, P.wait_budget);
                const volatile uint32_t* there_words = reinterpret_cast<const volatile uint32_t*>(smem + C::kOffWords) + 4 * w;
                const uint32_t words[4] = {there_words[0], there_words[1], there_words[2], there_words[3]};
                ok = ok && mbar_wait(bar_s + 8 * half, mine & 1, abort_flag, P.wait_budget);
                ++mine;
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                auto bits_of = [&](int pc) {                     // the row's columns of 32 from 32 pc on
                    const int t0 = base + 32 * pc;
                    const uint32_t word = pc == 0 ? words[0] : pc == 1 ? words[1] : pc == 2 ? words[2] : words[3];
                    return low_bits(tq - t0 + 1) & ~(tq - t0 >= A.K ? low_bits(tq - t0 - A.K + 1) : 0u) & word;
                };
                if (__any_sync(0xffffffffu, m == -CUDART_INF_F)) {
#pragma unroll 1
                    for (int pc = 0; pc < 4; ++pc) {             // rows that meet their first columns: their maximum
                        const uint32_t bits = bits_of(pc);
                        if (!__any_sync(0xffffffffu, m == -CUDART_INF_F && bits != 0u)) continue;
                        uint32_t s[32];
                        tmem_ld32(scol + 32 * pc, s);
                        const float by = landed(A.scale_log2);
                        float top = -CUDART_INF_F;
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if ((bits >> i) & 1u) top = fmaxf(top, __fmul_rn(__uint_as_float(s[i]), by));
                        if (m == -CUDART_INF_F) {
                            m = top;
                            if (fabsf(top) >= kFar && top != -CUDART_INF_F) limit = -1.f;
                        }
                    }
                }
                // A tile that every row of the warp sees all of (most of a long context): no masks, and the probabilities stay in
                // registers until the tile's sum has told that none of them outgrew its maximum.
                bool stored = false;
                if ((words[0] & words[1] & words[2] & words[3]) == 0xffffffffu && base + kKeys - 1 <= t_least && t_most - base < A.K &&
                    !__any_sync(0xffffffffu, m == -CUDART_INF_F)) {
                    uint32_t s[4][32], pk[4][16];                // two pieces ahead: all four at once would spill
                    const uint64_t nb2 = pack2(-m, -m);
                    uint64_t sum0 = 0ull, sum1 = 0ull;
                    tmem_ld32(scol, s[0]);
                    tmem_ld32(scol + 32, s[1]);
                    uint64_t by2 = landed(sc2);
#pragma unroll
                    for (int pc = 0; pc < 4; ++pc) {
                        if (pc < 2) tmem_ld32(scol + 32 * (pc + 2), s[pc + 2]);
                        uint32_t(&x)[32] = s[pc];
#pragma unroll
                        for (int i = 0; i < 16; i += 2) {
                            const uint64_t e = fma2(pack2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), by2, nb2);
                            const uint64_t g = fma2(pack2(__uint_as_float(x[2 * i + 2]), __uint_as_float(x[2 * i + 3])), by2, nb2);
                            float a = 0.f, b = 0.f;
                            if (i % 6 == 0) exp2_fma(e, a, b);
                            else {
                                a = fast_exp2(lo_of(e));
                                b = fast_exp2(hi_of(e));
                            }
                            const float c = fast_exp2(lo_of(g)), d = fast_exp2(hi_of(g));
                            sum0 = add2(sum0, pack2(a, b));
                            sum1 = add2(sum1, pack2(c, d));
                            pk[pc][i] = cvt_pack<BF16>(a, b);
                            pk[pc][i + 1] = cvt_pack<BF16>(c, d);
                        }
                        if (pc < 2) by2 = landed(by2);
                    }
                    sum0 = add2(sum0, sum1);
                    const float rs = lo_of(sum0) + hi_of(sum0);
                    if (!__any_sync(0xffffffffu, !(rs <= limit))) {
                        l += rs;
                        stored = true;
#pragma unroll
                        for (int pc = 0; pc < 4; ++pc) tmem_st16(scol + 16 * pc, pk[pc]);
                    }
                }
                // Other tiles, 64 columns at a time.
                if (!stored) {
#pragma unroll 1
                    for (int hc = 0; hc < 2; ++hc) {
                        const uint32_t lo = bits_of(2 * hc), hi = bits_of(2 * hc + 1);
                        uint32_t pk[2][16];
                        if (!__any_sync(0xffffffffu, (lo | hi) != 0u)) {         // no row of the warp sees any of them
#pragma unroll
                            for (int i = 0; i < 16; ++i) pk[0][i] = 0u;
                            tmem_st16(scol + 32 * hc, pk[0]);
                            tmem_st16(scol + 32 * hc + 16, pk[0]);
                            continue;
                        }
                        const float base_m = m == -CUDART_INF_F ? 0.f : m;
                        uint32_t s[2][32];
                        tmem_ld32(scol + 64 * hc, s[0]);
                        tmem_ld32(scol + 64 * hc + 32, s[1]);
                        const uint64_t by2 = landed(sc2), nb2 = pack2(-base_m, -base_m);
                        float sum_a = 0.f, sum_b = 0.f;
#pragma unroll
                        for (int w2 = 0; w2 < 2; ++w2) {
                            const uint32_t bits = w2 ? hi : lo;
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const uint64_t e = fma2(pack2(__uint_as_float(s[w2][2 * i]), __uint_as_float(s[w2][2 * i + 1])), by2, nb2);
                                // whatever a hidden score gave
                                const float a = (bits >> (2 * i)) & 1u ? fast_exp2(lo_of(e)) : 0.f;
                                const float b = (bits >> (2 * i + 1)) & 1u ? fast_exp2(hi_of(e)) : 0.f;
                                sum_a += a;
                                sum_b += b;
                                pk[w2][i] = cvt_pack<BF16>(a, b);
                            }
                        }
                        const float rs = sum_a + sum_b;
                        if (__builtin_expect(!__any_sync(0xffffffffu, !(rs <= limit)), 1)) {
                            l += rs;
                            tmem_st16(scol + 32 * hc, pk[0]);    // over columns of this thread's that have been read
                            tmem_st16(scol + 32 * hc + 16, pk[1]);
                            continue;
                        }
                        // Rare: a score has outgrown the row's maximum (or is not a number), or the maximum is far from zero.  16 columns
                        // at a time, from TMEM again.
                        auto exponents = [&](int q, uint32_t (&e)[16], float from) {     // (scaled scores, from = 0)
                            tmem_ld16(scol + 64 * hc + 16 * q, e);
                            const float by = landed(A.scale_log2);
                            const uint32_t bits = (q < 2 ? lo : hi) >> (16 * (q & 1));
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                e[i] = __float_as_uint((bits >> i) & 1u ? __fsub_rn(__fmul_rn(__uint_as_float(e[i]), by), from) : -CUDART_INF_F);
                        };
                        float top = -CUDART_INF_F;
#pragma unroll 1
                        for (int q = 0; q < 4; ++q) {
                            uint32_t e[16];
                            exponents(q, e, 0.f);
#pragma unroll
                            for (int i = 0; i < 16; ++i) top = fmaxf(top, __uint_as_float(e[i]));
                        }
                        const bool grow = top - base_m > kGrow;
                        if (__any_sync(0xffffffffu, grow)) rescale(grow, top, had_tiles, 2 * hc);
                        const float from = m == -CUDART_INF_F ? 0.f : m;
#pragma unroll 1
                        for (int q = 0; q < 4; ++q) {
                            uint32_t e[16], w8[8];
                            exponents(q, e, from);
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const float a = fast_exp2(__uint_as_float(e[2 * i])), b = fast_exp2(__uint_as_float(e[2 * i + 1]));
                                l += a + b;
                                w8[i] = cvt_pack<BF16>(a, b);
                            }
                            tmem_st8(scol + 32 * hc + 8 * q, w8);
                        }
                    }
                }
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive(bar_p + 8 * half);
                had_tiles = true;
            }
            if (!ok) break;

            // ---- output ----
            float f_mine = 1.f, f_other = 0.f;
            if (n > 0) {
                if (SPLIT && half == 1) {
                    if (exchanges > 0) ok = ok && warp_wait(bar_sums + 8, (exchanges - 1) & 1, abort_flag, P.wait_budget);
                    if (!ok) break;
                    sums[(warp & 3) * 32 + lane] = make_float2(m, l);
                    mbar_arrive(bar_sums);
                    ++exchanges;
                    ++units;
                    continue;                                    // the first half writes the rows
                }
                if (SPLIT && n > 1) {
                    ok = warp_wait(bar_sums, exchanges & 1, abort_flag, P.wait_budget) && ok;
                    ok = ok && warp_wait(bar_o + 8, exchanges & 1, abort_flag, P.wait_budget);
                    if (!ok) break;
                    const float2 other = sums[(warp & 3) * 32 + lane];
                    mbar_arrive(bar_sums + 8);
                    ++exchanges;
                    const float top = fmaxf(m, other.x), base_m = top == -CUDART_INF_F ? 0.f : top;
                    f_mine = fast_exp2(m - base_m);
                    f_other = fast_exp2(other.x - base_m);
                    l = l * f_mine + other.y * f_other;
                    m = top;
                }
                ok = ok && warp_wait(bar_o + 8 * half, units & 1, abort_flag, P.wait_budget);
                if (!ok) break;
                tc_fence_after();
            }
            const bool some = live && l != 0.f;                  // (a NaN stays one)
            float inv = direct ? (some ? 1.f / l : 0.f) : 1.f;
            const bool both = SPLIT && n > 1;
            // Four lanes exchange 16-byte pieces, so that a store writes 64 bytes of each of eight rows.
            long long rows4[4];
            const long long my_row = direct ? index : in_tile ? row : -1;
#pragma unroll
            for (int i = 0; i < 4; ++i) rows4[i] = __shfl_sync(0xffffffffu, my_row, (lane & ~3) | i);
            const int piece4 = lane & 3;
            constexpr int kPartsAtOnce = SPLIT ? 1 : DH / 32;    // (joining two halves, the code is too long to unroll)
#pragma unroll kPartsAtOnce
            for (int part = 0; part < DH / 32; ++part) {
                uint32_t o[32];
                if (n > 0) {
                    tmem_ld32(ocol + 32 * part, o);
                    if (both) {
                        uint32_t y[32];
                        tmem_ld32(trow + kColO + 128 + 32 * part, y);
                        const uint64_t mine2 = landed(pack2(f_mine, f_mine)), other2 = pack2(f_other, f_other);
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const uint64_t z = fma2(pack2(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1])), mine2,
                                                    tcplan::mul2(pack2(__uint_as_float(y[2 * i]), __uint_as_float(y[2 * i + 1])), other2));
                            o[2 * i] = __float_as_uint(lo_of(z));
                            o[2 * i + 1] = __float_as_uint(hi_of(z));
                        }
                    }
                    inv = landed(inv);
                }
                if (direct) {
                    uint32_t y[4][4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            y[i][k] = some ? cvt_pack<BF16>(__uint_as_float(o[8 * i + 2 * k]) * inv, __uint_as_float(o[8 * i + 2 * k + 1]) * inv) : 0u;
                    transpose4(y, piece4);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (rows4[i] >= 0)
                            reinterpret_cast<uint4*>(static_cast<uint16_t*>(A.out) + rows4[i] * DH)[4 * part + piece4] =
                                make_uint4(y[i][0], y[i][1], y[i][2], y[i][3]);
                } else {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t y[4][4];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int k = 0; k < 4; ++k) y[i][k] = __float_as_uint(__uint_as_float(o[16 * h + 4 * i + k]) * inv);    // (times 1)
                        transpose4(y, piece4);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (rows4[i] >= 0)
                                reinterpret_cast<uint4*>(slot_out(A, where) + rows4[i] * DH)[8 * part + 4 * h + piece4] =
                                    make_uint4(y[i][0], y[i][1], y[i][2], y[i][3]);
                    }
                }
            }
            if (in_tile) {
                if (!direct) slot_sums(A, where)[row] = make_float2(live ? m : -CUDART_INF_F, live ? l : 0.f);
                else if (A.lse) A.lse[index] = some ? (m + log2f(l)) * 0.6931471805599453f : -CUDART_INF_F;
            }
            if (n > 0) {
                tc_fence_before();
                mbar_arrive(bar_ofree + 8 * half);
                if (both) mbar_arrive(bar_ofree + 8);
                ++units;
            }
        }
    }

    if (*abort_flag) abort_grace_sleep();
    tc_fence_before();
    __syncthreads();
    if (warp == 12) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
        if (lane == 0 && *abort_flag) tcplan::raise_status(P);
    }
}

} // namespace

// Keys of a cache, 64 channels of one head: [64, slot, block of 64 channels, head, page]; a box is `run` slots.
static bool encode_cache(CUtensorMap* map, const Args& A, bool bf16, const void* cache, const int64_t (&strides)[3], int run)
{
    const cuuint64_t dims[5] = {64, (cuuint64_t)A.page_size, (cuuint64_t)A.D / 64, (cuuint64_t)A.Hkv, (cuuint64_t)A.pages};
    const cuuint64_t bytes[4] = {(cuuint64_t)strides[1] * 2, 128, (cuuint64_t)strides[2] * 2, (cuuint64_t)strides[0] * 2};
    const cuuint32_t box[5] = {64, (cuuint32_t)run, 1, 1, 1}, steps[5] = {1, 1, 1, 1, 1};
    return tcplan::encode_16bit(map, cache, bf16, dims, bytes, box, steps);
}

// Queries, 64 channels: [64, head, token, block of 64 channels, sequence]; a box is the rows of a tile, the heads of a group first.
static bool encode_queries(CUtensorMap* map, const Args& A, bool bf16)
{
    const cuuint64_t dims[5] = {64, (cuuint64_t)A.Hq, (cuuint64_t)A.L, (cuuint64_t)A.D / 64, (cuuint64_t)A.B};
    const cuuint64_t bytes[4] = {(cuuint64_t)A.qs[2] * 2, (cuuint64_t)A.qs[1] * 2, 128, (cuuint64_t)A.qs[0] * 2};
    const cuuint32_t box[5] = {64, (cuuint32_t)A.G, (cuuint32_t)(A.M / A.G), 1, 1}, steps[5] = {1, 1, 1, 1, 1};
    return tcplan::encode_16bit(map, A.q, bf16, dims, bytes, box, steps);
}

bool tc_shape(int dtype, const Args& A, bool aligned, Shape& shape)
{
    if ((dtype != NATTEN_F16 && dtype != NATTEN_BF16) || !aligned || (A.D != 64 && A.D != 128)) return false;
    const long long rows = ((long long)A.L + A.dil - 1) / A.dil * A.G;
    // 36 rows a unit over a context of 8192 (16 sequences): 76 us here, 149 on the other kernel; 64 rows over 8192 (8 sequences) 52 | 84.
    // A short context goes the other way (64 rows of 64 channels over 1024, 32 sequences: 32 | 25).  Its length is on the device; of the
    // bound that the host has, window and table (`divide`), this rule makes no use.
    if (rows <= 32) return false;
    shape = {rows > kHalfRows ? 2 * kHalfRows : kHalfRows, kKeys, 1, 2, 8, sm_count()};
    return true;
}

int tc_run(int dtype, const Args& call, cudaStream_t s)
{
    Args A = call;
    Status st{};
    st.wait_budget = tcplan::debug_wait_budget();
    st.inject = tcplan::debug_inject();
    cudaError_t err = tcplan::status_ptr(st.status);
    if (err == cudaSuccess) err = tcplan::status_host_ptr(st.status_host);
    if (err != cudaSuccess) return (int)err;
    // Runs of 64, 32 or 16 adjacent keys where the page size is a multiple of that many and nothing is dilated.
    CUtensorMap mq{}, mk{}, mv{};
    if (A.dil == 1 && A.pages > 0 && A.page_size % 16 == 0) {
        const int run = A.page_size % 64 == 0 ? 64 : A.page_size % 32 == 0 ? 32 : 16;
        if (encode_cache(&mk, A, dtype == NATTEN_BF16, A.kc, A.ks, run) && encode_cache(&mv, A, dtype == NATTEN_BF16, A.vc, A.vs, run)) A.align = run;
    }
    st.boxed = A.dil == 1 && A.M % A.G == 0 && encode_queries(&mq, A, dtype == NATTEN_BF16);
    auto go = [&](auto dh, auto bf, auto split) {
        constexpr int kDim = decltype(dh)::value;
        using C = Cfg<kDim, decltype(split)::value>;
        auto* kernel = tc_kernel<kDim, decltype(bf)::value, decltype(split)::value>;
        err = ensure_dynamic_smem((const void*)kernel, C::kSmem);
        if (err == cudaSuccess) kernel<<<A.ctas, kThreads, C::kSmem, s>>>(mq, mk, mv, A, st);
    };
    auto by_rows = [&](auto dh, auto bf) {
        if (A.M == kHalfRows) go(dh, bf, std::true_type{});
        else go(dh, bf, std::false_type{});
    };
    auto by_dim = [&](auto bf) {
        if (A.D == 64) by_rows(std::integral_constant<int, 64>{}, bf);
        else by_rows(std::integral_constant<int, 128>{}, bf);
    };
    if (dtype == NATTEN_BF16) by_dim(std::true_type{});
    else by_dim(std::false_type{});
    if (err == cudaSuccess) err = cudaGetLastError();
    tc_count_launch();
    return (int)err;
}

} // namespace paged
} // namespace natten
