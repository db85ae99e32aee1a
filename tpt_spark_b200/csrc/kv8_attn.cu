// kv8_attn.cu -- attention of one query row per sequence over the paged 8-bit KV cache.
//
// For key j of block (page, kv head) with scales ks, vs and codes c, d:
//     s_j = (q . c_j) ks / sqrt(hd),     out = sum_j softmax(s)_j vs d_j.
// S runs on the 8-bit integer tensor cores against the codes as they lie in memory: a query is written as
// q = step (256 a + b) (f32: step (65536 a + 256 b + c)) with signed 8-bit digits, so the sums are
// exact and q is off by at most 2^-16 (f32: 2^-23) of its largest element.  O needs weights of
// any size and runs in fp16, where codes are exact too; each scale multiplies a 16-key tile's scores and
// weights.
//
// Bound: every K and V byte is read once for the whole head group (HBM); close behind it the instructions per tile (the
// codes of V become fp16 by byte permutes onto 1024 + 128 + c).  The layout is built around bytes in flight and
// few instructions: 16 keys are the M of one tensor-core step, so the 8 columns carry up to 8 query heads,
//     S^T[key][head] = K . Q^T,          O^T[dim][head] += V^T . P^T,
// (a larger group reads its keys once for every 8)
// and the k indices of S and the dims of O are permuted so that each thread needs whole 16-byte
// runs of the codes.  Each warp has a ring of its own (cp.async, whole runs of a page: copies that took 32 bytes
// of a row at a time moved 1.5 times the bytes from L2), so the loop has no barrier: a warp waits for its copies only.
//
// Work split: the 16-key tiles of all (sequence, kv head) pairs form one line, cut into equal
// ranges, one per CTA, so ragged batches are balanced whatever the lengths; inside a range the
// warps take every kWarps-th tile.  A pair that several CTAs share is joined by the last of them (a
// ticket per pair), adding the parts in CTA order: results do not depend on scheduling.
//
// Weights: p = 2^(x - m) with a reference m that moves only when a score passes it by 8 (f32 sum
// l).  The tensor core takes p vs 2^-r as fp16, where m + r is the same kind of reference for
// x + log2 vs: pages whose scales differ by any ratio keep fp16's relative precision against the
// largest contribution.  For f32 the weights go in as a high and a low fp16 part.  (r is held by itself and
// scores are compared by their differences: with m around 2^27 a sum has steps of 16.)
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "serve.h"

namespace tptc {

namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kStages = 3;
constexpr int kCtasPerSm = 3;  // (4, with 128 registers and 2 stages: 98 us for 8 sequences of 32k against 87)
constexpr int kTile = 16;       // keys
constexpr int kHeads = 8;       // query heads per pass over the keys (columns of the products)
constexpr int kBlock = 128;     // parts whose weights are in shared memory at a time
// Units that make a CTA worth its share of the join (8: 777 positions take 9.8 us instead of 10.4; 32: they take 13.7,
// and one sequence of 16384 takes 17.6 instead of 18.8; batches that fill the GPU do not notice).
constexpr int kMinTiles = 16;
// A pair's place on the line: kSetup units for its queries and its join, then its tiles.  (With tiles alone, ranges
// of many short sequences took longest: 74 us instead of 52 for 32 sequences of 40 to 8000 positions; 8 or 32 units: 53.)
constexpr int kSetup = 16;

template <int HD>
struct Lay {
    static constexpr int kKVec = HD == 96 ? 8 : 16;   // bytes of a run of K
    static constexpr int kKPer = HD / 4 / kKVec;      // runs per row and thread
    static constexpr int kVVec = HD == 128 ? 16 : HD == 96 ? 4 : 8;
    static constexpr int kVPer = HD / 8 / kVVec;
    static constexpr int kKBytes = kTile * HD;
    static constexpr int kStage = 2 * kKBytes;
    static constexpr int kRing = kWarps * kStages * kStage;
    static constexpr int kRecord = 3 * kHeads + kHeads * HD;  // floats: m, l, r, O of one part
    // the warps' records, later the weights of a block of parts and their references
    static constexpr int kJoinA = kWarps * kRecord * 4, kJoinB = (2 * kBlock * kHeads + kThreads * 2) * 4;
    static constexpr int kJoin = kJoinA > kJoinB ? kJoinA : kJoinB;
    static constexpr int kSmem = kRing + kJoin;
};

__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

template <int BYTES>
__device__ __forceinline__ void lds(uint32_t (&w)[BYTES / 4], uint32_t addr) {
    if constexpr (BYTES == 16)
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr) : "memory");
    else if constexpr (BYTES == 8)
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr) : "memory");
    else
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(addr) : "memory");
}

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Bytes 0, 1 (HI: 2, 3) of a word of codes + 128 as fp16 codes: 1024 + byte is exact, so is the difference.
template <bool HI>
__device__ __forceinline__ uint32_t codes2(uint32_t w) {
    const uint32_t h = __byte_perm(w, 0x64646464u, HI ? 0x4342 : 0x4140);
    const uint32_t off = 0x64806480u;  // 1152, 1152
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), *reinterpret_cast<const __half2*>(&off));
    return *reinterpret_cast<const uint32_t*>(&r);
}

template <typename T>
__device__ __forceinline__ void store4(T* p, float a, float b, float c, float d) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
    else *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(a, b), pack2<T>(c, d));
}

// a / b of numbers that are not negative; 32-bit where both fit.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    if (((a | b) >> 32) == 0) return (uint32_t)a / (uint32_t)b;
    return a / b;
}

struct Params {
    tptc_kv8 c;
    const void* q;
    int64_t q_stride;
    const int32_t* len;
    int n_heads;
    void* out;
    int* counters;   // [n_seq * pairs per sequence], zero between calls
    float* records;  // [2 * grid]
    float scale_log2;
};

// Length of a sequence (0: nothing, or out of range).
__device__ __forceinline__ int length_of(const Params& p, int b, bool report) {
    const int n = p.len[b];
    if (n < 0 || n > p.c.max_pages * p.c.page) {
        if (report && p.c.status) atomicExch(p.c.status, TPTC_ERR_ARG);
        return 0;
    }
    return n;
}

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) kv8_attn_kernel(const __grid_constant__ Params p) {
    using L = Lay<HD>;
    constexpr bool kSplit = sizeof(T) == 4;  // high and low parts
    constexpr int MT = HD / 16;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int s_scan[kWarps], s_start[3];
    __shared__ int s_last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    const int G = p.n_heads / p.c.n_kv, subs = (G + kHeads - 1) / kHeads, pairs = p.c.n_kv * subs;

    // ---- this CTA's range of the line
    auto units_of = [&](int b, bool report) {
        const int t = b < p.c.n_seq ? (length_of(p, b, report) + kTile - 1) / kTile : 0;
        return t ? t + kSetup : 0;
    };
    const int units0 = units_of(tid, blockIdx.x == 0);  // of the first kThreads sequences
    int64_t total = 0;
    for (int b0 = 0; b0 < p.c.n_seq; b0 += kThreads) {
        const int t = warp_sum_i(b0 == 0 ? units0 : units_of(b0 + tid, blockIdx.x == 0));
        if (b0 > 0) __syncthreads();
        if (lane == 0) s_scan[warp] = t;
        __syncthreads();
        for (int w = 0; w < kWarps; w++) total += s_scan[w];
    }
    // sequences without a position: zeros
    for (int b = blockIdx.x; b < p.c.n_seq; b += gridDim.x)
        if (length_of(p, b, false) == 0)
            for (int i = tid; i < p.n_heads * HD; i += kThreads)
                static_cast<T*>(p.out)[(int64_t)b * p.n_heads * HD + i] = static_cast<T>(0.f);
    total *= pairs;
    const int ctas = (int)min((int64_t)gridDim.x, (total + kMinTiles - 1) / kMinTiles);
    if ((int)blockIdx.x >= ctas) return;
    // CTA c begins at c share + min(c, more)
    const int64_t share = quotient(total, ctas);
    const int more = (int)(total - share * ctas);
    auto begins = [&](int c) { return c * share + min(c, more); };
    auto cta_of = [&](int64_t t) {  // whose range holds unit t
        const int64_t split = (share + 1) * more;
        return t < split ? (int)quotient(t, share + 1) : more + (int)quotient(t - split, share);
    };
    const int64_t first = begins(blockIdx.x), end = begins(blockIdx.x + 1);
    {
        int64_t before = 0;  // units before the block of sequences
        bool found = false;
        for (int b0 = 0; b0 < p.c.n_seq && !found; b0 += kThreads) {
            const int b = b0 + tid, t = b0 == 0 ? units0 : units_of(b, false);
            int incl = t;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
            }
            if (p.c.n_seq > kThreads) {  // (the warps' sums are still there when one block holds all sequences)
                __syncthreads();
                if (lane == 31) s_scan[warp] = incl;
                __syncthreads();
            }
            int64_t lead = before;
            for (int w = 0; w < warp; w++) lead += s_scan[w];
            const int64_t lo = (lead + incl - t) * pairs, hi = (lead + incl) * pairs;
            const bool mine = t > 0 && lo <= first && first < hi;
            if (mine) {
                s_start[0] = b;
                s_start[1] = (int)quotient(first - lo, t);
                s_start[2] = (int)(first - lo) - s_start[1] * t;
            }
            found = __syncthreads_or(mine);
            for (int w = 0; w < kWarps; w++) before += s_scan[w];
        }
    }
    int b = s_start[0], pair = s_start[1], tile = max(0, s_start[2] - kSetup);
    int len = length_of(p, b, false), tiles = (len + kTile - 1) / kTile;
    int64_t piece0 = first - s_start[2];  // the pair's first unit
    if (end - piece0 <= kSetup) return;   // not a tile

    const uint32_t ring = smem_u32(smem) + warp * (kStages * L::kStage);
    // Where a lane's copies go in a stage (512 bytes per copy of the warp, rows in order), and where a thread
    // finds its runs: 16-byte chunks change places inside 128 bytes so that both are free of bank conflicts.
    // K: rows g and g + 8; V: rows 2 t4 and 2 t4 + 1, and those behind them by 8.
    uint32_t k_to = lane * 16, v_to = lane * 16, k_of, v_of;
    if constexpr (HD == 128) {
        k_to = ((lane & ~7) | ((lane & 7) ^ ((lane & 8) >> 1))) * 16;
        v_to = ((lane & ~7) | ((lane & 7) ^ ((lane & 16) >> 3))) * 16;
        k_of = g * 128 + (t4 ^ ((g & 1) << 2)) * 16;
        v_of = t4 * 256 + (g ^ (t4 << 1)) * 16;
    } else if constexpr (HD == 64) {
        v_to = ((lane & ~7) | ((lane & 7) ^ ((lane & 24) >> 2))) * 16;
        k_of = g * 64 + t4 * 16;
        v_of = t4 * 128 + ((g >> 1) ^ (t4 << 1)) * 16 + (g & 1) * 8;
    } else {
        k_of = g * 96 + t4 * 8;
        v_of = t4 * 192 + g * 12;
    }
    auto k_run = [&](int r, int j) { return r * 8 * HD + (HD == 128 ? k_of ^ (j * 64) : k_of + j * 32); };
    auto v_run = [&](int r, int j) {
        return (r >> 1) * 8 * HD + (HD == 64 ? v_of ^ ((r & 1) * 64) : v_of + (r & 1) * HD + j * L::kVVec);
    };

    float* rec = reinterpret_cast<float*>(smem + L::kRing);  // the joins' memory
    auto ratio = [](float a, float m) { return a == m ? 1.f : ex2(a - m); };
    auto join_refs = [](float& m, float& r, float m2, float r2) {  // (NaN, of two that are empty, loses to any number)
        const float mn = fmaxf(m, m2);
        r = fmaxf(r + (m - mn), r2 + (m2 - mn));
        m = mn;
    };

    // ---- a piece: the CTA's part of one pair's tiles
    int n, kvh, h0, nh, mine;  // its tiles; heads; tiles of this warp
    int id0, id1, batch;       // page ids and scales: lane i holds those of the warp's tile 32 batch + i, and of the next batch
    float ks0, vs0, ks1, vs1;
    const int8_t *k_at, *v_at;
    constexpr int WORDS = HD / 16;  // of four dims
    using Four = typename std::conditional<kSplit, float4, uint2>::type;
    Four q_raw[WORDS];
    const int page_mask = p.c.page - 1;
    const int64_t page_bytes = (int64_t)p.c.n_kv * p.c.page * HD;  // of all heads
    auto fetch = [&](int of, int& id, float& ks, float& vs) {
        const int i = 32 * of + lane;
        id = 0;
        ks = vs = 0.f;
        if (i < mine) {
            const int pos = (tile + warp + i * kWarps) * kTile;
            id = p.c.table[(int64_t)b * p.c.max_pages + pos / p.c.page];
            if (id >= 0 && id < p.c.n_pages) {
                const int64_t k = (int64_t)id * p.c.n_kv + kvh;
                ks = p.c.k_scale[k];
                vs = p.c.v_scale[k];
            } else {  // not in the cache: not followed
                if (p.c.status) atomicExch(p.c.status, TPTC_ERR_ARG);
                id = 0;
                ks = vs = __int_as_float(0x7fc00000);
            }
        }
    };
    auto issue = [&](int i, int slot) {  // 2 x 16 rows, each a run of the page
        if (i < mine) {
            const int id = __shfl_sync(0xffffffffu, (i >> 5) == batch ? id0 : id1, i & 31);
            const int64_t off = id * page_bytes + (((tile + warp + i * kWarps) * kTile) & page_mask) * HD;
            const int8_t *k = k_at + off, *v = v_at + off;
            const uint32_t kd = ring + slot * L::kStage, vd = kd + L::kKBytes;
#pragma unroll
            for (int e = 0; e < HD / 32; e++) {
                copy_async(kd + e * 512 + k_to, k + e * 512);
                copy_async(vd + e * 512 + (HD == 128 && (e & 1) ? v_to ^ 64 : v_to), v + e * 512);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto begin = [&] {  // everything of it that can be on its way
        n = (int)min((int64_t)tiles, end - piece0 - kSetup) - tile;
        kvh = pair / subs;
        h0 = kvh * G + (pair % subs) * kHeads;
        nh = min(kHeads, kvh * G + G - h0);
        mine = n > warp ? (n - warp + kWarps - 1) / kWarps : 0;
        batch = 0;
        fetch(0, id0, ks0, vs0);
        fetch(1, id1, ks1, vs1);
        k_at = p.c.k + (int64_t)kvh * p.c.page * HD + lane * 16;
        v_at = p.c.v + (int64_t)kvh * p.c.page * HD + lane * 16;
        const T* q = static_cast<const T*>(p.q) + (int64_t)b * p.q_stride + (int64_t)(h0 + g) * HD;
#pragma unroll
        for (int w = 0; w < WORDS; w++) {
            constexpr int per = L::kKVec / 4;  // words per run
            q_raw[w] = Four{};
            if (g < nh) q_raw[w] = __ldg(reinterpret_cast<const Four*>(q + (w / per) * (4 * L::kKVec) + t4 * L::kKVec + (w % per) * 4));
        }
#pragma unroll
        for (int i = 0; i < kStages - 1; i++) issue(i, i);
    };

    begin();
    for (;;) {
        // ---- the queries, as the B operand: thread holds the digits of head g, dims of its own bytes of K
        constexpr int DIGITS = kSplit ? 3 : 2;
        uint32_t qd[DIGITS][WORDS];
        float fq0, fq1;
        {
            // the largest magnitude, as its bits (inf and NaN are above all numbers)
            uint32_t most = 0;
#pragma unroll
            for (int w = 0; w < WORDS; w++) {
                const uint32_t* raw = reinterpret_cast<const uint32_t*>(&q_raw[w]);
#pragma unroll
                for (int e = 0; e < (int)sizeof(T); e++)
                    most = kSplit ? max(most, raw[e] & 0x7fffffffu) : __vmaxu2(most, raw[e] & 0x7fff7fffu);
            }
            if constexpr (!kSplit) most = max(most & 0xffffu, most >> 16);
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
            const float top = kSplit ? __uint_as_float(most)
                              : std::is_same<T, __half>::value ? __half2float(__ushort_as_half((unsigned short)most))
                                                               : __uint_as_float(most << 16);
            // the largest element becomes 127 in its highest digit (a power of two first, so that no factor
            // leaves f32's range); an element that is not finite makes the head's scores NaN
            const int e2 = max(-126, min(126, (int)(__float_as_uint(top) >> 23) - 126));
            constexpr float kMost = kSplit ? 127.f * 65536.f : 127.f * 256.f;
            const float down = __uint_as_float((uint32_t)(127 - e2) << 23), unit = top * down;
            const float up = unit > 0.f ? __fdividef(kMost, unit) : 0.f;
#pragma unroll
            for (int s = 0; s < WORDS; s++) {
                uint32_t v[4];
                auto pack = [&](uint32_t byte) {  // byte 0 or 1 of each
                    const uint32_t sel = byte | (byte + 4) << 4;
                    return __byte_perm(__byte_perm(v[0], v[1], sel), __byte_perm(v[2], v[3], sel), 0x5410);
                };
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float x = to_f32(reinterpret_cast<const T*>(&q_raw[s])[e]) * down;
                    // (two digits fit the low half of 1.5 2^23 + v; conversions have a quarter of the rate)
                    if constexpr (kSplit) v[e] = (uint32_t)__float2int_rn(x * up);
                    else v[e] = __float_as_uint(fmaf(x, up, 12582912.f));
                }
                qd[DIGITS - 1][s] = pack(0);
                // the next digit is signed as well: (v - digit) / 256 = (v + 128) >> 8
#pragma unroll
                for (int d = DIGITS - 2; d >= 0; d--) {
#pragma unroll
                    for (int e = 0; e < 4; e++) v[e] += 128;
                    qd[d][s] = pack(1);
                    if (d > 0)
#pragma unroll
                        for (int e = 0; e < 4; e++) v[e] = (uint32_t)((int)v[e] >> 8);
                }
            }
            const float f = top <= 3.402823466e38f ? p.scale_log2 * (unit * (1.f / kMost)) * __uint_as_float((uint32_t)(127 + e2) << 23)
                                                   : __int_as_float(0x7fc00000);
            fq0 = __shfl_sync(0xffffffffu, f, 8 * t4);
            fq1 = __shfl_sync(0xffffffffu, f, 8 * t4 + 4);
        }

        float o[MT][4];
#pragma unroll
        for (int j = 0; j < MT; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;             // heads 2 t4 and 2 t4 + 1
        float r0 = -INFINITY, r1 = -INFINITY, w0 = INFINITY, w1 = INFINITY;  // r, and 2^-r
        int slot = 0;
        for (int i = 0; i < mine; i++) {
            if ((i >> 5) != batch) {
                batch++;
                id0 = id1, ks0 = ks1, vs0 = vs1;
                fetch(batch + 1, id1, ks1, vs1);
            }
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
            const float ks = __shfl_sync(0xffffffffu, ks0, i & 31), vs = __shfl_sync(0xffffffffu, vs0, i & 31);
            __syncwarp();  // the other lanes' copies; and every lane is through with the stage before
            const uint32_t k_from = ring + slot * L::kStage, v_from = k_from + L::kKBytes;

            // S^T: rows g and g + 8 are keys
            float s[4];
            {
                uint32_t a[WORDS], c[WORDS];
#pragma unroll
                for (int j = 0; j < L::kKPer; j++) {
                    lds<L::kKVec>(reinterpret_cast<uint32_t(&)[L::kKVec / 4]>(a[j * (L::kKVec / 4)]), k_from + k_run(0, j));
                    lds<L::kKVec>(reinterpret_cast<uint32_t(&)[L::kKVec / 4]>(c[j * (L::kKVec / 4)]),
                                  k_from + k_run(1, j));
                }
                // (a chain of products for each digit: they run side by side; 128 products of 127 by 127 are below 2^21)
                int d[DIGITS][4];
#pragma unroll
                for (int n = 0; n < DIGITS; n++) d[n][0] = d[n][1] = d[n][2] = d[n][3] = 0;
#pragma unroll
                for (int e = 0; e < WORDS; e += 2)
#pragma unroll
                    for (int n = 0; n < DIGITS; n++) mma_s8(d[n], a[e], c[e], a[e + 1], c[e + 1], qd[n][e], qd[n][e + 1]);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    s[e] = (float)(d[0][e] * 256 + d[1][e]);
                    if constexpr (kSplit) s[e] = fmaf(s[e], 256.f, (float)d[DIGITS - 1][e]);
                }
            }
            const float g0 = ks * fq0, g1 = ks * fq1;
            float x0 = s[0] * g0, x1 = s[1] * g1, x2 = s[2] * g0, x3 = s[3] * g1;
            const int key = (tile + warp + i * kWarps) * kTile;
            if (key + kTile > len) {  // the sequence's last tile
                if (key + g >= len) x0 = x1 = -INFINITY;
                if (key + g + 8 >= len) x2 = x3 = -INFINITY;
            }
            const float t0 = fmaxf(x0, x2), t1 = fmaxf(x1, x3);
            // (a NaN score never moves a reference; it reaches l and O below)
            float v0 = vs * w0, v1 = vs * w1;  // at most 2^7, so that weights stay below 2^15
            if (__any_sync(0xffffffffu, t0 - m0 > 8.f || t1 - m1 > 8.f || !(v0 <= 128.f) || !(v1 <= 128.f))) {
                float c0 = t0, c1 = t1;
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) {
                    c0 = fmaxf(c0, __shfl_xor_sync(0xffffffffu, c0, d));
                    c1 = fmaxf(c1, __shfl_xor_sync(0xffffffffu, c1, d));
                }
                // (log2 of a scale of zero or below the normal range would be -inf, and its weights inf or NaN)
                const float lv = lg2(fmaxf(vs, 1.17549435e-38f));
                auto move = [&](float c, float& m, float& l, float& r, float& w, float& v) {
                    const float mn = fmaxf(m, c), down = m == mn ? 0.f : m - mn;
                    const float was = r + down, rn = fmaxf(was, c - mn + lv);
                    l *= ex2(down);
                    const float beta = was == rn ? 1.f : ex2(was - rn);
                    m = mn, r = rn;
                    w = ex2(fminf(-rn, 127.f));
                    v = vs * w;
                    return beta;
                };
                const float b0 = move(c0, m0, l0, r0, w0, v0), b1 = move(c1, m1, l1, r1, w1, v1);
#pragma unroll
                for (int j = 0; j < MT; j++) o[j][0] *= b0, o[j][1] *= b1, o[j][2] *= b0, o[j][3] *= b1;
            }
            const float p0 = ex2(x0 - m0), p1 = ex2(x1 - m1), p2 = ex2(x2 - m0), p3 = ex2(x3 - m1);
            l0 += p0 + p2;
            l1 += p1 + p3;
            // The product takes 16-bit weights.  fp16, whatever the queries' type: 2^-11 each, below a bf16 output's own
            // 2^-8; the sum l takes them unrounded, as the roundings of many keys average out.
            uint32_t bh[2], bl[2];
            {
                const float y0 = p0 * v0, y1 = p1 * v1, y2 = p2 * v0, y3 = p3 * v1;
                const uint32_t ha = pack2<__half>(y0, y1), hb = pack2<__half>(y2, y3);
                bh[0] = transpose8x8(ha);
                bh[1] = transpose8x8(hb);
                if constexpr (kSplit) {
                    const float2 fa = __half22float2(*reinterpret_cast<const __half2*>(&ha));
                    const float2 fb = __half22float2(*reinterpret_cast<const __half2*>(&hb));
                    bl[0] = transpose8x8(pack2<__half>(y0 - fa.x, y1 - fa.y));
                    bl[1] = transpose8x8(pack2<__half>(y2 - fb.x, y3 - fb.y));
                }
            }
            // O^T: rows g and g + 8 of step j are dims 2 j and 2 j + 1 of the thread's bytes
#pragma unroll
            for (int j = 0; j < L::kVPer; j++) {
                uint32_t v[4][L::kVVec / 4];
#pragma unroll
                for (int r = 0; r < 4; r++) lds<L::kVVec>(v[r], v_from + v_run(r, j));
#pragma unroll
                for (int e = 0; e < L::kVVec / 4; e++) {
                    // keys 2 t4 and 2 t4 + 1 (+ 8) beside one another, dims 0 1 | 2 3
                    uint32_t ab0 = __byte_perm(v[0][e], v[1][e], 0x5140) ^ 0x80808080u;
                    uint32_t ab1 = __byte_perm(v[0][e], v[1][e], 0x7362) ^ 0x80808080u;
                    uint32_t cd0 = __byte_perm(v[2][e], v[3][e], 0x5140) ^ 0x80808080u;
                    uint32_t cd1 = __byte_perm(v[2][e], v[3][e], 0x7362) ^ 0x80808080u;
                    const uint32_t f0[4] = {codes2<false>(ab0), codes2<true>(ab0), codes2<false>(cd0), codes2<true>(cd0)};
                    const uint32_t f1[4] = {codes2<false>(ab1), codes2<true>(ab1), codes2<false>(cd1), codes2<true>(cd1)};
                    const int k = 2 * (j * (L::kVVec / 4) + e);
                    mma(o[k], f0, bh[0], bh[1]);
                    mma(o[k + 1], f1, bh[0], bh[1]);
                    if constexpr (kSplit) {
                        mma(o[k], f0, bl[0], bl[1]);
                        mma(o[k + 1], f1, bl[0], bl[1]);
                    }
                }
            }
            issue(i + kStages - 1, slot == 0 ? kStages - 1 : slot - 1);
            slot = slot == kStages - 1 ? 0 : slot + 1;
        }
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
            l0 += __shfl_xor_sync(0xffffffffu, l0, d);
            l1 += __shfl_xor_sync(0xffffffffu, l1, d);
        }

        // ---- the next piece's copies run under this one's join
        const int was_n = n, was_h = nh, was_tiles = tiles;
        const int64_t was0 = piece0, was1 = piece0 + kSetup + tiles;  // the pair's part of the line
        T* out = static_cast<T*>(p.out) + ((int64_t)b * p.n_heads + h0) * HD;
        int* counter = p.counters + (int64_t)b * pairs + pair;
        const bool again = end - was1 > kSetup;
        if (again) {
            piece0 = was1;
            tile = 0;
            if (++pair == pairs) {
                pair = 0;
                do len = length_of(p, ++b, false);
                while (len == 0);  // (a sequence with tiles follows: the range goes on)
                tiles = (len + kTile - 1) / kTile;
            }
            __syncwarp();  // every lane is through with the ring
            begin();
        }

        // ---- join the warps
        __syncthreads();  // the last join's memory is free
        {
            float* me = rec + warp * L::kRecord;
            if (g == 0) {
                me[2 * t4] = m0, me[2 * t4 + 1] = m1;
                me[kHeads + 2 * t4] = l0, me[kHeads + 2 * t4 + 1] = l1;
                me[2 * kHeads + 2 * t4] = r0, me[2 * kHeads + 2 * t4 + 1] = r1;
            }
            float* mo = me + 3 * kHeads;
#pragma unroll
            for (int j = 0; j < MT; j++) {
                float* a = mo + (2 * t4) * HD + g * (HD / 8) + 2 * j;
                *reinterpret_cast<float2*>(a) = make_float2(o[j][0], o[j][2]);
                *reinterpret_cast<float2*>(a + HD) = make_float2(o[j][1], o[j][3]);
            }
        }
        __syncthreads();
        const bool whole = was_n == was_tiles;
        // slot 0 of the CTA: a pair that began before its range; 1: one that begins inside it
        float* out_rec = p.records + (int64_t)(2 * blockIdx.x + (first >= was0 ? 0 : 1)) * L::kRecord;
        // a thread holds four dims of a head per step; parts are scaled to the largest references
        for (int i = tid; i < kHeads * (HD / 4); i += kThreads) {
            const int h = i / (HD / 4), d = (i % (HD / 4)) * 4;
            float m = -INFINITY, r = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; w++) m = fmaxf(m, rec[w * L::kRecord + h]);
#pragma unroll
            for (int w = 0; w < kWarps; w++) r = fmaxf(r, rec[w * L::kRecord + 2 * kHeads + h] + (rec[w * L::kRecord + h] - m));
            float l = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < kWarps; w++) {
                const float* a = rec + w * L::kRecord;
                if (w >= was_n) break;  // a warp without a tile
                l += a[kHeads + h] * ratio(a[h], m);
                const float f = ratio(a[2 * kHeads + h] + (a[h] - m), r);
                const float4 v = *reinterpret_cast<const float4*>(a + 3 * kHeads + h * HD + d);
                y[0] += v.x * f, y[1] += v.y * f, y[2] += v.z * f, y[3] += v.w * f;
            }
            if (whole) {
                const float f = ex2(r) / l;
                if (h < was_h) store4(out + h * HD + d, y[0] * f, y[1] * f, y[2] * f, y[3] * f);
            } else {
                if (d == 0) out_rec[h] = m, out_rec[kHeads + h] = l, out_rec[2 * kHeads + h] = r;
                *reinterpret_cast<float4*>(out_rec + 3 * kHeads + h * HD + d) = make_float4(y[0], y[1], y[2], y[3]);
            }
        }
        if (!whole) {
            const int c0 = cta_of(was0 + kSetup), c1 = cta_of(was1 - 1), parts = c1 - c0 + 1;
            __syncthreads();
            if (tid == 0) {  // the release covers this CTA's record, the last one's acquire all of them
                int n_before;
                asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(n_before) : "l"(counter) : "memory");
                s_last = n_before == parts - 1;
                if (s_last) *counter = 0;
            }
            __syncthreads();
            if (s_last) {
                // (only the first part's CTA can have begun before the pair)
                const float* parts_at = p.records + 2 * (int64_t)c0 * L::kRecord;
                const int first_off = begins(c0) >= was0 ? 0 : L::kRecord;
                auto part = [&](int i) { return parts_at + (i == 0 ? first_off : i * (2 * L::kRecord)); };
                // the references of all parts, 16 parts of 8 heads at a time
                constexpr int kRows = kThreads / kHeads;
                float *w_l = rec, *w_o = rec + kBlock * kHeads, *ref = rec + 2 * kBlock * kHeads;
                const int h8 = tid % kHeads, k8 = tid / kHeads;
                {
                    float m = -INFINITY, r = -INFINITY;
#pragma unroll 4
                    for (int k = k8; k < parts; k += kRows) {
                        const float* a = part(k);
                        join_refs(m, r, __ldcg(a + h8), __ldcg(a + 2 * kHeads + h8));
                    }
                    ref[k8 * 2 * kHeads + h8] = m;
                    ref[k8 * 2 * kHeads + kHeads + h8] = r;
                }
                __syncthreads();
                float m_all = -INFINITY, r_all = -INFINITY;  // of head h8
                for (int k = 0; k < kRows; k++)
                    join_refs(m_all, r_all, ref[k * 2 * kHeads + h8], ref[k * 2 * kHeads + kHeads + h8]);
                constexpr int kSteps = (kHeads * (HD / 4) + kThreads - 1) / kThreads;
                float l[kSteps], y[kSteps][4];
#pragma unroll
                for (int e = 0; e < kSteps; e++) l[e] = y[e][0] = y[e][1] = y[e][2] = y[e][3] = 0.f;
                for (int k0 = 0; k0 < parts; k0 += kBlock) {
                    const int count = min(kBlock, parts - k0);
                    __syncthreads();
                    for (int k = k8; k < count; k += kRows) {
                        const float* a = part(k0 + k);
                        const float m = __ldcg(a + h8);
                        w_l[k * kHeads + h8] = __ldcg(a + kHeads + h8) * ratio(m, m_all);
                        w_o[k * kHeads + h8] = ratio(__ldcg(a + 2 * kHeads + h8) + (m - m_all), r_all);
                    }
                    __syncthreads();
#pragma unroll
                    for (int e = 0; e < kSteps; e++) {
                        const int i = tid + e * kThreads, h = i / (HD / 4), d = (i % (HD / 4)) * 4;
                        if (h >= was_h) continue;
#pragma unroll 8
                        for (int k = 0; k < count; k++) {
                            const float f = w_o[k * kHeads + h];
                            const float4 v = __ldcg(reinterpret_cast<const float4*>(part(k0 + k) + 3 * kHeads + h * HD + d));
                            l[e] += w_l[k * kHeads + h];
                            y[e][0] += v.x * f, y[e][1] += v.y * f, y[e][2] += v.z * f, y[e][3] += v.w * f;
                        }
                    }
                }
                if (k8 == 0) ref[h8] = ex2(r_all);
                __syncthreads();
#pragma unroll
                for (int e = 0; e < kSteps; e++) {
                    const int i = tid + e * kThreads, h = i / (HD / 4), d = (i % (HD / 4)) * 4;
                    if (h >= was_h) continue;
                    const float f = ref[h] / l[e];
                    store4(out + h * HD + d, y[e][0] * f, y[e][1] * f, y[e][2] * f, y[e][3] * f);
                }
            }
        }
        if (!again) break;
    }
}

int grid_of(int sms) { return kCtasPerSm * sms; }
int pairs_of(int n_heads, int n_kv) { return n_kv * ceil_div(n_heads / n_kv, kHeads); }
// The records lie first, in room for the widest heads, and the counters behind them: a workspace that has served
// one shape holds zero counters for every other that fits it.
size_t record_bytes(int sms) { return (size_t)2 * grid_of(sms) * Lay<128>::kRecord * sizeof(float); }

template <typename T, int HD>
cudaError_t launch(const Params& p, int sms, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid_of(sms));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Lay<HD>::kSmem;
    cfg.stream = st;
    return cudaLaunchKernelEx(&cfg, kv8_attn_kernel<T, HD>, p);
}

template <typename T>
cudaError_t launch_t(const Params& p, int sms, cudaStream_t st) {
    if (p.c.head_dim == 64) return launch<T, 64>(p, sms, st);
    if (p.c.head_dim == 96) return launch<T, 96>(p, sms, st);
    return launch<T, 128>(p, sms, st);
}

template <typename T>
cudaError_t init_t() {
    cudaError_t e = cudaFuncSetAttribute(kv8_attn_kernel<T, 64>, cudaFuncAttributeMaxDynamicSharedMemorySize, Lay<64>::kSmem);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(kv8_attn_kernel<T, 96>, cudaFuncAttributeMaxDynamicSharedMemorySize, Lay<96>::kSmem);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(kv8_attn_kernel<T, 128>, cudaFuncAttributeMaxDynamicSharedMemorySize, Lay<128>::kSmem);
    return e;
}

}  // namespace

// A warp adds the units of up to 32 sequences in 32 bits.
bool kv8_attn_fits(const tptc_kv8& c) {
    const int64_t most = (int64_t)c.max_pages * c.page / kTile + kSetup;
    return std::min(c.n_seq, 32) * most <= INT32_MAX;
}

size_t kv8_attn_workspace(const tptc_kv8& c, int n_heads, int sms) {
    return record_bytes(sms) + (size_t)c.n_seq * pairs_of(n_heads, c.n_kv) * sizeof(int);
}

cudaError_t launch_kv8_attn(int type, const Kv8Attn& a, int sms, cudaStream_t st) {
    Params p = {};
    p.c = a.c;
    p.q = a.q;
    p.q_stride = a.q_stride;
    p.len = a.len;
    p.n_heads = a.n_heads;
    p.out = a.out;
    p.records = reinterpret_cast<float*>(a.workspace);
    p.counters = reinterpret_cast<int*>(a.workspace + record_bytes(sms));
    p.scale_log2 = (float)(1.4426950408889634 / sqrt((double)a.c.head_dim));
    if (type == TPTC_TYPE_F16) return launch_t<__half>(p, sms, st);
    if (type == TPTC_TYPE_BF16) return launch_t<__nv_bfloat16>(p, sms, st);
    return launch_t<float>(p, sms, st);
}

cudaError_t kv8_attn_init_device() {
    cudaError_t e = init_t<__half>();
    if (e == cudaSuccess) e = init_t<__nv_bfloat16>();
    if (e == cudaSuccess) e = init_t<float>();
    return e;
}

}  // namespace tptc
