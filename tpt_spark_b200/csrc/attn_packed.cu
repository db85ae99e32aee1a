// attn_packed.cu -- causal attention over packed prompts of different lengths (tcgen05).
//
// Query i of a sequence with lq queries and lk keys sees keys 0 .. lk - lq + i.  For head h of
// the group of kv head h / G:  S = Q K^T / sqrt(hd),  O = softmax(S) V.
//
// Tile: 128 TMEM lanes hold floor(128 / G) consecutive tokens x the G heads of one kv head, so every
// lane is in use for short prompts too and a K/V tile is shared by the whole group.  A CTA owns two
// such tiles, A and B, which stream the same tiles of K and V through one ring, each with its own
// issuing warp and its own softmax warpgroup.
// TMEM holds for both tiles the scores S (BN columns), the weights P as 16-bit pairs (BN / 2) and O (HD):
// with P beside S and not in its place, the scores of the next keys are computed while the
// exponentials of these run.  BN is what then fits 512 columns (128, 96, 80 keys for head_dim 64, 96,
// 128).  P enters its product from TMEM.
// A lane stores its own row at the end, 32 bytes at a time.  (Whole lines by way of shared memory: 105 us became 120 for
// 12 prompts of 60 to 2100 tokens with 64-wide heads.)
// Bounds, per pair of tiles and 128 keys at head_dim 128: 2048 cycles of exponentials (16 per cycle and
// SM) and 2350 of the tensor core (S waits for shared memory, 6.5 KB of operands per 40 cycles).  What is
// reached is 3450: a lone softmax warp's chain of waits, loads, maximum, exponentials and stores.
// Tried and slower, at the time: two threads per lane (519 us for 8192 tokens, 32 heads on 8, against 441), a quarter of the exponentials
// as polynomials (483 against 462), P in the place of S with 128 keys per tile (448), turns of A
// and B at the exponentials (470).
// Measured there: 445 us = 1235 TFLOP/s in single calls, 517 us back to back (the power limit lowers the clock).
//
// Softmax: one thread per lane, base 2, with a reference maximum that moves (rescaling O in TMEM and
// the f32 sum) only when a tile's maximum passes it by 8, so P stays below 2^8.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "serve.h"
#include "tcgen05.cuh"

namespace tptc {

namespace {

constexpr int BM = 128;
constexpr int kThreads = 384;  // warpgroup 0: copies (warp 0), products of A and B (1, 2), items (3); 1 and 2: their softmax
// Registers: 384 threads launch with 168 each; the softmax threads hold 128 scores and take what
// warpgroup 0 gives back (128 x (72 + 2 x 216) = 384 x 168).
constexpr int kRegsFew = 72, kRegsMany = 216;
constexpr int kTmemCols = 512;

template <int HD>
struct Lay {
    static constexpr int BN = HD == 64 ? 128 : HD == 96 ? 96 : 80;  // keys per tile
    // Weights handed over at once, then the rest.  (head_dim 128, 8192 tokens: all 80 at once 441 us, 32, 48 or 64 first 467.)
    static constexpr int kFirst = HD == 128 ? 80 : 64;
    static constexpr int kP = 2 * BN, kO = 3 * BN;     // TMEM columns: S_A, S_B from 0, P_A, P_B, O_A, O_B
    static constexpr int NC = (HD + 63) / 64;          // 64-column blocks of a row (the last may be part empty)
    static constexpr int kQTile = BM * NC * 128;       // bytes of a tile of Q
    static constexpr int kTile = BN * NC * 128;        // of K or V
    static constexpr int kStages = (220 * 1024 - 2 * kQTile) / kTile < 8 ? (220 * 1024 - 2 * kQTile) / kTile : 8;
    static constexpr int kKV = 2 * kQTile;
    static constexpr int kBytes = kKV + kStages * kTile;
    static_assert(kO + 2 * HD <= kTmemCols && kTile % 1024 == 0 && kStages >= 5, "layout");
};

struct Params {
    void* out;
    const int32_t *cu_q, *cu_k;
    int n_seq, n_q, n_k, max_q, n_heads, n_kv;
    int tokens;  // per tile
    uint32_t pair_mul, pair_shift;  // n / (2 tokens) = n pair_mul >> 32 >> pair_shift for n below 2^31
    float scale_log2;
    int32_t* status;
};

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::
            "r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
        : "memory");
}

// D += A B with A in TMEM.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
        "r"(a), "l"(bdesc), "r"(idesc), "r"(acc)
        : "memory");
}

// Waits for a phase of a barrier; false when it does not come (a bounded number
// of polls) or when another wait of the CTA gave up.  One instruction and a branch where the phase is complete:
// the loops of this kernel wait up to ten times per tile, and with a called-out abort flag and a vote in each
// wait 8192 tokens took 523 us instead of 463; the flag is read behind a poll that failed.  Such a poll sleeps
// for 4 us (measured), so that waiting warps leave the issue slots to the others, and the limit is 17 s: the longest
// wait is one item, and the keys that fit the memory take 10.
constexpr uint32_t kPolls = 1u << 22;
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, const uint32_t* gave_up) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n .reg .u32 n, g;\n mov.u32 n, %3;\n"
        "POLL:\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %4;\n @p bra DONE;\n"
        " sub.u32 n, n, 1;\n ld.volatile.shared.u32 g, [%5];\n setp.eq.u32 p, n, 0;\n setp.ne.or.u32 p, g, 0, p;\n @!p bra POLL;\n"
        " setp.lt.u32 p, n, 0;\n"
        "DONE:\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "n"(kPolls), "r"(10000), "r"(smem_u32(gave_up))
        : "memory");
    return ok != 0;
}
// The same for what writes to this CTA's memory or reads it, and so has to end before the CTA does, whoever gave up.
__device__ __forceinline__ bool wait_own(uint64_t* bar, uint32_t parity) {
    for (uint32_t n = 0; n < kPolls; n++)
        if (mbar_try_wait(bar, parity)) return true;
    return false;
}

// One lane of a converged warp.  (The compiler keeps what a warp computes alike in uniform registers, where
// the products' operands have to be; under `lane == 0` each product cost about 100 cycles to issue.)
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.b32 %0, 1, 0, p;\n}\n" : "=r"(one));
    return one != 0;
}

// N columns, not waited for; tmem_loads_done() ends the wait for all loads before it.
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, float* r) {
    static_assert(N == 16 || N == 32, "columns");
    if constexpr (N == 16)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                     : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
                     : "r"(taddr));
    if constexpr (N == 32)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                     : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
                     : "r"(taddr));
}
__device__ __forceinline__ void tmem_loads_done() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// Keeps the uses of loaded registers behind the wait.
__device__ __forceinline__ void pin16(float* r) {
    asm volatile("" : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]),
                 "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15]));
}
template <int N>
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t* r) {
    static_assert(N == 8 || N == 16 || N == 32, "columns");
    if constexpr (N == 8)
        asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
    if constexpr (N == 16)
        asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
    if constexpr (N == 32)
        asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
// N columns, a multiple of 8.
template <int N>
__device__ __forceinline__ void store_p(uint32_t taddr, const uint32_t* r) {
    if constexpr (N >= 32) {
        tmem_st<32>(taddr, r);
        if constexpr (N > 32) store_p<N - 32>(taddr + 32, r + 32);
    } else if constexpr (N >= 16) {
        tmem_st<16>(taddr, r);
        if constexpr (N > 16) store_p<N - 16>(taddr + 16, r + 16);
    } else {
        tmem_st<8>(taddr, r);
    }
}
__device__ __forceinline__ void tmem_stores_done() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// A reference m is the largest score times scale_log2, rounded; what the rounding cut off (up to |m| 2^-24) shifts every
// exponent of the lane alike and cancels.  For scores of billions (q and k around 60000 in fp16) it would take
// the weights out of the type's range, so a lane whose m passes kFar subtracts the reference from the
// scores themselves, exactly.  (All lanes always: 113 us instead of 102 for 12 prompts of 60 to 2100 tokens; this rare branch: 103.)
constexpr float kFar = 65536.f;

// 32 bytes of a row (a whole sector) in one store.
__device__ __forceinline__ void store32(void* p, const uint32_t* r) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// Two f32 fused multiply-adds or sums in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)),
          "l"(reinterpret_cast<const unsigned long long&>(c)));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)));
    return d;
}

// ---- work items.  A CTA that is through with its own block index takes over that of a CTA that has not
// started yet (cluster launch control), so that TMEM, barriers and the ring are set up once per SM, the next
// item's loads run under the current one's last products, and the hardware balances ragged batches.

__device__ __forceinline__ void request_item(uint4* response, uint64_t* bar) {
    mbar_expect_tx(bar, 16);
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                     smem_u32(response)),
                 "r"(smem_u32(bar))
                 : "memory");
}
// Block indices: x is the kv head, y and z the place in the list of pairs of tiles (no division on the way).
constexpr int kPlacesY = 32768;
struct Place {
    int kvh, k;  // k -1: none
};
// The block index taken over, if one was left.
__device__ __forceinline__ Place taken_place(const uint4* response) {
    uint32_t x, y, z, got;
    asm volatile(
        "{\n .reg .pred p;\n .reg .b128 r;\n ld.shared.b128 r, [%4];\n"
        " clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n selp.u32 %3, 1, 0, p;\n"
        " mov.u32 %0, 0;\n mov.u32 %1, 0;\n mov.u32 %2, 0;\n"
        " @p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%0, %1, %2, _}, r;\n}\n"
        : "=&r"(x), "=&r"(y), "=&r"(z), "=&r"(got)
        : "r"(smem_u32(response))
        : "memory");
    return {(int)x, got ? (int)(y + z * kPlacesY) : -1};
}

struct Rows {
    int q_lo, q_hi, k_lo, k_hi;
};
__device__ __forceinline__ Rows rows_of(const Params& p, int b) { return {p.cu_q[b], p.cu_q[b + 1], p.cu_k[b], p.cu_k[b + 1]}; }
// Pairs of tiles that a sequence has; 0 where there is nothing to do or its offsets are out of range.
__device__ __forceinline__ int pairs_of(const Params& p, const Rows& r, bool report) {
    if (r.q_lo == r.q_hi) return 0;
    if (r.q_lo < 0 || r.q_hi < r.q_lo || r.q_hi > p.n_q || r.q_hi - r.q_lo > p.max_q || r.k_lo < 0 || r.k_hi < r.k_lo || r.k_hi > p.n_k) {
        if (report && p.status) atomicExch(p.status, TPTC_ERR_ARG);
        return 0;
    }
    return (int)(__umulhi((uint32_t)(r.q_hi - r.q_lo - 1), p.pair_mul) >> p.pair_shift) + 1;
}

struct alignas(16) Item {
    int q0, k0;     // packed rows: the first token of tile A, the sequence's first key
    int base, lk;   // tile A's first token sees base + 1 keys; keys of the sequence
    int toks[2], nt[2];  // tokens of a tile, and the key tiles that its last token sees
    int kvh, ntot;  // ntot -1: no more items
};

// The list of items, walked by one warp: the places are ordered by level, then by sequence, where the
// level is the number of a pair of tiles in its sequence, from the highest down: those with the most keys come first,
// and nothing is launched for pairs that a short sequence does not have.  (With n_seq x longest indices,
// 63 prompts of one token beside one of 8192 took 836 us instead of 452.)
constexpr int kSeqs = 2048;  // sequences whose counts are kept in shared memory
struct List {
    const int* counts;  // [kSeqs]
    int top;            // pairs of the longest sequence
    int lo, hi;         // levels that the same sequences have (`count` of them): hi - 1 down to lo
    int64_t before;     // the first place of level hi - 1 (places: items of a kv head)
    int count;
    int level, b0, skipped;  // of the last item found: its level, block of 32 sequences, and sequences before those
    __device__ __forceinline__ int pairs(const Params& p, int b) const {
        return b < p.n_seq ? (b < kSeqs ? counts[b] : pairs_of(p, rows_of(p, b), false)) : 0;
    }
    __device__ __forceinline__ void levels_below(const Params& p, int top) {  // hi = top
        hi = top;
        count = 0;
        int next = 0;
        for (int b = 0; b < p.n_seq; b += 32) {
            const int n = pairs(p, b + (threadIdx.x & 31));
            count += __popc(__ballot_sync(0xffffffffu, n >= hi));
            next = max(next, n < hi ? n : 0);
        }
        lo = __reduce_max_sync(0xffffffffu, next);
    }
    // sequence of place k, and its level; false: behind the last.  (Places ascend: what was found before is the start.)
    __device__ __forceinline__ bool find(const Params& p, int k, int& b) {
        if (p.n_seq == 1) {  // (a level has one place)
            b = 0;
            level = top - 1 - k;
            return level >= 0;
        }
        if (hi == 0 || k < before) {
            if (top == 0) return false;
            before = 0;
            levels_below(p, top);
        }
        while (k - before >= (int64_t)(hi - lo) * count) {
            if (lo == 0) return false;
            before += (int64_t)(hi - lo) * count;
            levels_below(p, lo);
        }
        const int at_k = (int)(k - before), down = at_k / count, r = at_k - down * count, lane = threadIdx.x & 31;
        if (hi - 1 - down != level || r < skipped) level = hi - 1 - down, b0 = skipped = 0;
        for (; b0 < p.n_seq; b0 += 32) {
            const bool has = pairs(p, b0 + lane) > level;
            const uint32_t m = __ballot_sync(0xffffffffu, has);
            const uint32_t at = __ballot_sync(0xffffffffu, has && skipped + __popc(m & ((1u << lane) - 1)) == r);
            if (at) {
                b = b0 + __ffs(at) - 1;
                return true;
            }
            skipped += __popc(m);
        }
        return false;
    }
};
template <int BN>
__device__ __forceinline__ Item item_of(const Params& p, const Rows& r, int pair, int kvh) {
    const int lq = r.q_hi - r.q_lo, lk = r.k_hi - r.k_lo, tok0 = pair * 2 * p.tokens;
    Item w;
    w.q0 = r.q_lo + tok0;
    w.k0 = r.k_lo;
    w.kvh = kvh;
    w.lk = lk;
    w.base = lk - lq + tok0;
#pragma unroll
    for (int t = 0; t < 2; t++) {
        w.toks[t] = max(0, min(p.tokens, lq - tok0 - t * p.tokens));
        const int sees = w.base + t * p.tokens + w.toks[t];
        w.nt[t] = w.toks[t] > 0 && sees > 0 ? (sees + BN - 1) / BN : 0;
    }
    w.ntot = max(w.nt[0], w.nt[1]);
    return w;
}

constexpr int kLead = 4;  // key tiles of an item still to load when the next one is asked for

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, 1)
    attn_packed_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                       const __grid_constant__ CUtensorMap tv, const __grid_constant__ Params p) {
    using L = Lay<HD>;
    constexpr int S = L::kStages, KS = HD / 16, BN = L::BN;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t q_full, q_empty, full[S], empty[S], item_full[2], item_empty[2], wanted, taken;
    __shared__ uint64_t s_full[2], s_free[2], p_full[2][2], pv_done[2], drain[2];
    __shared__ uint4 response;
    __shared__ Item items[2];
    __shared__ int counts[kSeqs];
    __shared__ uint32_t tmem_slot, gave_up;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = p.n_heads / p.n_kv;

    if (threadIdx.x == 0) {
        gave_up = 0;
        mbar_init(&q_full, 1);
        mbar_init(&q_empty, 2);  // both tiles' products are through with it
        for (int s = 0; s < S; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 2);
        }
        for (int t = 0; t < 2; t++) {
            mbar_init(&s_full[t], 1);
            mbar_init(&s_free[t], 4);  // one arrival per softmax warp
            for (int h = 0; h < 2; h++) mbar_init(&p_full[t][h], 4);
            mbar_init(&pv_done[t], 1);
            mbar_init(&drain[t], 1);
            mbar_init(&item_full[t], 1);
            mbar_init(&item_empty[t], 11);  // copies, two product warps and eight softmax warps have read it
        }
        mbar_init(&wanted, 1);
        mbar_init(&taken, 1);
        fence_mbar_init();
    }
    if (warp == 1) tmem_alloc(&tmem_slot, kTmemCols);
    // The list's warp: the first item is there when the CTA starts.  (An index behind the list's end: an item of nothing.)
    List list = {counts, 0, 0, 0, 0, 0, -1, 0, 0};
    Rows known = {};  // of sequence `lane`, loaded once
    auto listed_item = [&](const Place& at, Item& w) {
        int b = 0;
        if (!list.find(p, at.k, b)) return false;
        Rows r;
        if (b < 32)
            r = {__shfl_sync(0xffffffffu, known.q_lo, b), __shfl_sync(0xffffffffu, known.q_hi, b),
                 __shfl_sync(0xffffffffu, known.k_lo, b), __shfl_sync(0xffffffffu, known.k_hi, b)};
        else
            r = rows_of(p, b);
        w = item_of<BN>(p, r, list.level, at.kvh);
        return true;
    };
    if (warp == 3) {
        for (int b = lane; b < p.n_seq; b += 32) {
            const Rows r = rows_of(p, b);
            const int n = pairs_of(p, r, blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0);
            if (b < 32) known = r;
            if (b < kSeqs) counts[b] = n;
            list.top = max(list.top, n);
        }
        list.top = __reduce_max_sync(0xffffffffu, list.top);
        __syncwarp();
        Item w = {};
        listed_item({(int)blockIdx.x, (int)(blockIdx.y + blockIdx.z * kPlacesY)}, w);
        if (lane == 0) items[0] = w;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    auto give_up = [&] {
        *reinterpret_cast<volatile uint32_t*>(&gave_up) = 1;
        if (p.status) atomicExch(p.status, TPTC_ERR_TIMEOUT);
        return false;
    };
    auto wait = [&](uint64_t* bar, uint32_t parity) { return wait_phase(bar, parity, &gave_up) || give_up(); };
    // the n-th item of the CTA, for a lane (copies) or a warp; false: no more
    auto get_item = [&](int n, Item& w, bool whole_warp) {
        const int s = n & 1;
        if (n > 0 && !wait(&item_full[s], (n >> 1) & 1)) return false;
        w = items[s];
        if (whole_warp) __syncwarp();
        if (!whole_warp || lane == 0) mbar_arrive(&item_empty[s]);
        return w.ntot >= 0;
    };

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsFew));
        if (warp == 0 && lane == 0) {  // copies: Q_A, Q_B, then K_0, V_0, K_1, ... of each item
            int i0 = 0, nq = 0;        // loads into the ring and Q tiles so far
            bool ok = true;
            Item w;
            for (int n = 0; ok && get_item(n, w, false); n++) {
                if (w.ntot <= kLead) mbar_arrive(&wanted);
                if (w.ntot == 0) continue;
                if (nq > 0) ok = mbar_wait_backoff(&q_empty, (nq - 1) & 1, nullptr) || give_up();
                if (!ok) break;
                nq++;
                mbar_expect_tx(&q_full, (w.toks[1] > 0 ? 2 : 1) * ((uint32_t)(p.tokens * G) * 128 * L::NC));
                for (int t = 0; t < 2; t++) {
                    if (w.toks[t] == 0) continue;
#pragma unroll
                    for (int c = 0; c < L::NC; c++)
                        tma_load_3d(smem + t * L::kQTile + c * BM * 128, &tq, c * 64, w.kvh * G, w.q0 + t * p.tokens, &q_full);
                }
                for (int k = 0; k < 2 * w.ntot; k++, i0++) {
                    const int s = i0 % S;
                    if (i0 >= S) ok = mbar_wait_backoff(&empty[s], ((i0 / S) - 1) & 1, nullptr) || give_up();
                    if (!ok) break;
                    mbar_expect_tx(&full[s], L::kTile);
#pragma unroll
                    for (int c = 0; c < L::NC; c++)
                        tma_load_3d(smem + L::kKV + s * L::kTile + c * BN * 128, (k & 1) ? &tv : &tk, c * 64, w.kvh,
                                    w.k0 + (k >> 1) * BN, &full[s]);
                    if (w.ntot > kLead && k == 2 * (w.ntot - kLead) - 1) mbar_arrive(&wanted);
                }
            }
            // the copies still in flight land before the CTA exits
            if (nq > 0) wait_own(&q_full, (nq - 1) & 1);
            for (int k = i0 > S ? i0 - S : 0; k < i0; k++) wait_own(&full[k % S], (k / S) & 1);
        }
        if (warp == 3) {  // the items behind the first, asked for when the copies of the one before near their end
            if (lane == 0) mbar_arrive(&item_full[0]);
            Place at = {0, 0};
            for (int n = 1, asked = 0; at.k >= 0; n++) {
                Item w = {};
                w.ntot = -1;
                at.k = -1;
                if (wait(&wanted, (n - 1) & 1)) do {  // (indices behind the list's end are taken over until none is left)
                    if (lane == 0) request_item(&response, &taken);
                    if (wait_own(&taken, asked++ & 1) || give_up()) at = taken_place(&response);
                    else at.k = -1;
                    fence_proxy_async_smem();  // read before the slot is written again
                    __syncwarp();
                } while (at.k >= 0 && !listed_item(at, w));
                const int s = n & 1;
                if (n >= 2 && !wait(&item_empty[s], ((n >> 1) - 1) & 1)) break;
                if (lane == 0) {
                    items[s] = w;
                    mbar_arrive(&item_full[s]);
                }
            }
        }
        if (warp == 1 || warp == 2) {  // products of a tile: the whole warp waits, one elected lane issues
            const int t = warp - 1;
            constexpr uint32_t type_bits = std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u;
            constexpr uint32_t id_s = mma_idesc(BM, BN) | type_bits, id_o = mma_idesc(BM, HD) | kIdescBMajorMN | type_bits;
            // (descriptors hold the address / 16 in their low bits: steps inside a tile are added there)
            const uint64_t q_desc = sw128_desc(smem_u32(smem + t * L::kQTile)), k_desc = sw128_desc(smem_u32(smem + L::kKV));
            const uint64_t v_desc = sw128_desc_mn(smem_u32(smem + L::kKV), BN * 128);
            const uint32_t tS = tmem + t * BN, tP = tmem + L::kP + t * (BN / 2), tO = tmem + L::kO + t * HD;
            const bool one = elect_one();
            int i0 = 0, nq = 0, ns = 0, np = 0;  // loads, Q tiles, scores and weights so far
            auto wait_full = [&](int i) { return wait(&full[i % S], (i / S) & 1); };
            auto commit = [&](uint64_t* bar) {
                if (one) mma_commit(bar);
            };
            auto issue_s = [&](int i) {  // i: the load of K; the last scores have been taken up
                if (ns > 0 && !wait(&s_free[t], (ns - 1) & 1)) return false;
                ns++;
                tc_fence_after();
                const uint64_t ka = k_desc + i % S * (L::kTile / 16);
                if (one) {
#pragma unroll
                    for (int k = 0; k < KS; k++)
                        mma_f16(tS, q_desc + ((k / 4) * BM * 128 + 32 * (k % 4)) / 16,
                                ka + ((k / 4) * BN * 128 + 32 * (k % 4)) / 16, id_s, k != 0);
                    mma_commit(&s_full[t]);
                }
                return true;
            };
            auto issue_pv = [&](int i, bool first) {  // i: the load of V; the weights come in two parts
                const uint64_t va = v_desc + i % S * (L::kTile / 16);
#pragma unroll
                for (int h = 0; h < (L::kFirst < BN ? 2 : 1); h++) {
                    if (!wait(&p_full[t][h], np & 1)) return false;
                    tc_fence_after();
                    if (one) {
#pragma unroll
                        for (int k = h ? L::kFirst / 16 : 0; k < (h ? BN : L::kFirst) / 16; k++)
                            mma_ts(tO, tP + 8 * k, va + k * (2048 / 16), id_o, !first || k != 0);
                    }
                }
                np++;
                commit(&pv_done[t]);
                return true;
            };
            bool ok = true;
            Item w;
            for (int n = 0; ok && get_item(n, w, true); n++) {
                if (w.ntot == 0) continue;
                const int nt = t ? w.nt[1] : w.nt[0];
                ok = wait(&q_full, nq & 1) && wait_full(i0);
                if (!ok) break;
                nq++;
                if (nt > 0) ok = issue_s(i0);
                commit(&empty[i0 % S]);
                if (w.ntot == 1) commit(&q_empty);
                for (int j = 0; j < w.ntot && ok; j++) {
                    const int iv = i0 + 2 * j + 1, ik = iv + 1;
                    if (j + 1 < w.ntot) {
                        ok = wait_full(ik);
                        if (ok && j + 1 < nt) ok = issue_s(ik);
                        if (!ok) break;
                        commit(&empty[ik % S]);
                        if (j + 2 == w.ntot) commit(&q_empty);
                    }
                    ok = wait_full(iv);
                    if (ok && j < nt) ok = issue_pv(iv, j == 0);
                    if (ok) commit(&empty[iv % S]);
                }
                i0 += 2 * w.ntot;
            }
            // every product issued has completed before TMEM is freed
            commit(&drain[t]);
            wait_own(&drain[t], 0);
            __syncwarp();
        }
    } else {  // one thread per lane of tile A or B
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsMany));
        const int t = (warp >> 2) - 1, r = 32 * (warp & 3) + lane;
        const uint32_t loff = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t tS = tmem + t * BN + loff, tP = tmem + L::kP + t * (BN / 2) + loff, tO = tmem + L::kO + t * HD + loff;
        int i0 = 0, ns = 0;  // loads and score tiles so far
        bool ok = true;
        Item w;
        for (int n = 0; get_item(n, w, true); n++) {
            const int nt = t ? w.nt[1] : w.nt[0], toks = t ? w.toks[1] : w.toks[0];
            const int tok = t * p.tokens + min(r / G, max(toks - 1, 0));  // spare lanes follow the last token
            const int sees = w.base + tok + 1, all_see = w.base + t * p.tokens + 1;  // keys of this lane, and of every lane
            // the reference is m, or the score `ref` where that is set (m is -inf then, and every tile "moves" it)
            float m = -INFINITY, l = 0.f, ref = -INFINITY;
            for (int j = 0; j < nt; j++, ns++) {
                ok = wait(&s_full[t], ns & 1);
                if (!ok) break;
                tc_fence_after();
                float s[BN];
#pragma unroll
                for (int c = 0; c + 32 <= BN; c += 32) tmem_ld<32>(tS + c, s + c);
                if constexpr (BN % 32 != 0) tmem_ld<16>(tS + BN / 32 * 32, s + BN / 32 * 32);
                tmem_loads_done();
#pragma unroll
                for (int c = 0; c < BN; c += 16) pin16(s + c);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&s_free[t]);
                if ((j + 1) * BN > all_see) {
                    const int left = sees - j * BN;
#pragma unroll
                    for (int k = 0; k < BN; k++) s[k] = k < left ? s[k] : -INFINITY;
                }
                float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int k = 4; k < BN; k += 8)
#pragma unroll
                    for (int c = 0; c < 4; c++) mx[c] = k + 4 + c < BN ? max3(mx[c], s[k + c], s[k + 4 + c]) : fmaxf(mx[c], s[k + c]);
                const float most = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), mt = most * p.scale_log2;
                const bool move = mt > m + 8.f;
                float alpha = 1.f;
                const float m_was = m;
                if (move) {
                    alpha = ex2(m - mt);
                    m = mt;
                }
                if (__builtin_expect(move && (fabsf(mt) > kFar || ref > -INFINITY), 0)) {
                    const float to = (most - ref) * p.scale_log2 > 8.f ? most : ref;  // (ref -inf: most)
                    alpha = ref == -INFINITY ? ex2(m_was - to * p.scale_log2) : to == ref ? 1.f : ex2((ref - to) * p.scale_log2);
                    m = -INFINITY;
                    ref = to;
#pragma unroll
                    for (int k = 0; k < BN; k++) s[k] -= ref;
                }
                if (move) l *= alpha;
                const float neg = m == -INFINITY ? 0.f : -m;  // a lane that sees nothing yet: weights 0
                const float2 sc = make_float2(p.scale_log2, p.scale_log2), off = make_float2(neg, neg);
                float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                uint32_t x[BN / 2];
                auto weights = [&](int k0, int k1) {
#pragma unroll
                    for (int k = k0; k < k1; k++) {
                        const float2 y = fma2(make_float2(s[2 * k], s[2 * k + 1]), sc, off);
                        const float2 e = make_float2(ex2(y.x), ex2(y.y));
                        sum[k & 1] = add2(sum[k & 1], e);
                        x[k] = pack2<T>(e.x, e.y);  // (the product takes 16 bits; the sum takes e, as many roundings average out)
                    }
                };
                auto hand_over = [&](int h) {
                    tmem_stores_done();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_full[t][h]);
                };
                weights(0, L::kFirst / 2);
                // the last product has taken up P and added to O
                if (j > 0) {
                    ok = wait(&pv_done[t], (ns - 1) & 1);
                    if (!ok) break;
                    tc_fence_after();
                    if (__any_sync(0xffffffffu, move)) {
#pragma unroll 1
                        for (int c = 0; c < HD; c += 32) {
                            float o[32];
                            uint32_t z[32];
                            tmem_ld<32>(tO + c, o);
                            tmem_loads_done();
                            pin16(o);
                            pin16(o + 16);
#pragma unroll
                            for (int i = 0; i < 32; i++) z[i] = __float_as_uint(o[i] * alpha);
                            tmem_st<32>(tO + c, z);
                        }
                    }
                }
                const int iv = i0 + 2 * j + 1;
                if ((j + 1) * BN > w.lk && wait(&full[iv % S], (iv / S) & 1)) {
                    // rows behind the sequence's last key may hold anything: zero them in V, so that
                    // weight 0 times them is 0 (both tiles write the same zeros, each before its product)
                    uint8_t* vb = smem + L::kKV + (iv % S) * L::kTile;
                    const int r0 = w.lk - j * BN, cnt = (BN - r0) * L::NC * 8;
                    for (int i = r; i < cnt; i += BM) {
                        const int row = r0 + i / (L::NC * 8), rem = i % (L::NC * 8);
                        *reinterpret_cast<uint4*>(vb + (rem >> 3) * BN * 128 + row * 128 + (rem & 7) * 16) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async_smem();
                }
                store_p<L::kFirst / 2>(tP, x);
                hand_over(0);
                if constexpr (L::kFirst < BN) {
                    weights(L::kFirst / 2, BN / 2);
                    store_p<(BN - L::kFirst) / 2>(tP + L::kFirst / 2, x + L::kFirst / 2);
                    hand_over(1);
                }
                sum[0] = add2(sum[0], sum[1]);
                l += sum[0].x + sum[0].y;
            }
            if (!ok) break;
            if (nt > 0) {
                ok = wait(&pv_done[t], (ns - 1) & 1);
                if (!ok) break;
                tc_fence_after();
            }
            if (toks > 0) {
                const float il = l > 0.f || l != l ? 1.f / l : 0.f;
                const bool mine = r < toks * G;
                T* row = static_cast<T*>(p.out) + ((int64_t)(w.q0 + tok) * p.n_heads + w.kvh * G + r % G) * HD;
#pragma unroll 1
                for (int c = 0; c < HD; c += 32) {
                    float o[32];
                    if (nt > 0) {
                        tmem_ld<32>(tO + c, o);
                        tmem_loads_done();
                        pin16(o);
                        pin16(o + 16);
                    }
                    if (mine) {
                        uint32_t z[16];
#pragma unroll
                        for (int i = 0; i < 16; i++) z[i] = il == 0.f ? 0u : pack2<T>(o[2 * i] * il, o[2 * i + 1] * il);
#pragma unroll
                        for (int i = 0; i < 16; i += 8) store32(row + c + 2 * i, z + i);
                    }
                }
            }
            i0 += 2 * w.ntot;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

template <typename T, int HD>
cudaError_t launch(const AttnPacked& a, Params p, cudaStream_t st) {
    const int G = a.n_heads / a.n_kv;
    CUtensorMap tq, tk, tv;
    const bool bf = std::is_same<T, __nv_bfloat16>::value;
    cudaError_t e = make_tmap_heads(&tq, a.q, bf, HD, a.n_heads, a.n_q, a.q_stride, G, p.tokens);
    if (e == cudaSuccess && a.n_k > 0) e = make_tmap_heads(&tk, a.k, bf, HD, a.n_kv, a.n_k, a.k_stride, 1, Lay<HD>::BN);
    if (e == cudaSuccess && a.n_k > 0) e = make_tmap_heads(&tv, a.v, bf, HD, a.n_kv, a.n_k, a.v_stride, 1, Lay<HD>::BN);
    if (e != cudaSuccess) return e;
    if (a.n_k == 0) tk = tv = tq;  // no key: no copy is made
    // pairs of tiles: no sequence has more than the longest, and together they have at most one that is not full each
    const int64_t pairs = std::min((int64_t)a.n_seq * ceil_div64(std::min(a.max_q, a.n_q), 2 * p.tokens),
                                   (int64_t)a.n_q / (2 * p.tokens) + a.n_seq);
    uint32_t log2 = 1;  // of 2 tokens, rounded up
    while ((1u << log2) < 2u * p.tokens) log2++;
    p.pair_mul = (uint32_t)(((1ull << (31 + log2)) + 2 * p.tokens - 1) / (2 * p.tokens));
    p.pair_shift = log2 - 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.n_kv, (unsigned)std::min(pairs, (int64_t)kPlacesY), (unsigned)ceil_div64(pairs, kPlacesY));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Lay<HD>::kBytes + 1024;
    cfg.stream = st;
    return cudaLaunchKernelEx(&cfg, attn_packed_kernel<T, HD>, tq, tk, tv, p);
}

template <typename T>
cudaError_t launch_t(const AttnPacked& a, const Params& p, cudaStream_t st) {
    if (a.head_dim == 64) return launch<T, 64>(a, p, st);
    if (a.head_dim == 96) return launch<T, 96>(a, p, st);
    return launch<T, 128>(a, p, st);
}

template <typename T>
cudaError_t init_t() {
    cudaError_t e = cudaFuncSetAttribute(attn_packed_kernel<T, 64>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         Lay<64>::kBytes + 1024);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(attn_packed_kernel<T, 96>, cudaFuncAttributeMaxDynamicSharedMemorySize, Lay<96>::kBytes + 1024);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(attn_packed_kernel<T, 128>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 Lay<128>::kBytes + 1024);
    return e;
}

}  // namespace

cudaError_t attn_packed_init_device() {
    cudaError_t e = init_t<__half>();
    if (e == cudaSuccess) e = init_t<__nv_bfloat16>();
    return e;
}

cudaError_t launch_attn_packed(int type, const AttnPacked& a, cudaStream_t st) {
    Params p = {};
    p.out = a.out;
    p.cu_q = a.cu_q;
    p.cu_k = a.cu_k;
    p.n_seq = a.n_seq;
    p.n_q = a.n_q;
    p.n_k = a.n_k;
    p.max_q = a.max_q;
    p.n_heads = a.n_heads;
    p.n_kv = a.n_kv;
    p.tokens = BM / (a.n_heads / a.n_kv);
    p.scale_log2 = (float)(1.4426950408889634 / sqrt((double)a.head_dim));
    p.status = a.status;
    if (type == TPTC_TYPE_F16) return launch_t<__half>(a, p, st);
    return launch_t<__nv_bfloat16>(a, p, st);
}

}  // namespace tptc
