// logprobs.cu -- log probabilities of given tokens, entropy and the largest alternatives of each
// row of logits, in one pass over the logits.
//
// With m = max x, z = sum e^(x - m) and t = sum e^(x - m) (x - m):
//     log p(i) = x_i - m - log z,      entropy = log z - t / z.
// A thread keeps (m, z, t) of its elements and moves them to a new maximum m' by
// z <- z a, t <- a (t + z (m - m')), a = e^(m - m'); the CTA's states join in thread order.
//
// The n largest, exactly and with ties by lowest index.  An element is one 64-bit key (ordered
// value bits, then ~index): keys are unique and their order is the wanted one.  Each warp keeps
// its n largest sorted, lane i the i-th, and looks at a chunk's elements again only when one of
// the threads' maxima of 16 elements (32 of 16 bits; the online maximum needs them anyway) reaches a threshold: the larger of
// the warp's own n-th, of the n-th largest of the first chunk's 32 group maxima, and of the r-th largest
// over the warps of their k-th, k r >= n, which they publish without a barrier (each bounds the
// row's n-th from below, whenever it is read).  About n ln(vocab / chunk) elements of a row are
// ever inserted.  (A shared candidate list with a barrier per chunk took 341 us for 1500 bf16 rows of 128256,
// this takes 88 us; both with n = 5.)
//
// One CTA per row streams the logits.  For 16-bit logits the instructions bound it (issue 64 %, exponentials 59 %;
// 1500 rows without the n largest take 71 us, 5.4 TB/s).  The sums are f32: a thread adds runs of 16 or 32 elements,
// then threads and warps join, so that a term meets few roundings (5e-8 off a sum in 64 bits for 128256 tokens).
// With few rows a cluster of CTAs shares one row and joins through distributed shared memory (latency bound).
#include <algorithm>
#include <type_traits>

#include "serve.h"

namespace tptc {

namespace {

constexpr int kThreads = 256;                // kWarps lists of up to 32 keys: also the cluster join's shape
constexpr int kVecs = 4;                     // 16-byte vectors per thread and chunk
constexpr int kWarps = kThreads / 32;
constexpr int kMaxParts = 8;
constexpr int kStages = 3;                   // chunks of the ring: two are on their way
constexpr int kCtasPerSm = 4;
constexpr int kRing = kStages * kVecs * kThreads * 16;

__device__ __forceinline__ uint32_t ordered(float x) {
    if (isnan(x)) return 0xffffffffu;
    x += 0.f;  // -0 equals 0
    const uint32_t u = __float_as_uint(x);
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t o) {
    if (o == 0xffffffffu) return __int_as_float(0x7fc00000);
    return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}

struct State {
    float m, z, t;
};
// The state of the disjoint sets of the first `lanes` lanes (a power of two), in every one of
// them; an empty set has m = -inf, z = t = 0.  The sums run in a fixed order.
__device__ __forceinline__ State join_lanes(State s, int lanes) {
    float m = s.m;
    for (int o = 1; o < lanes; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float d = s.m - m, w = s.z == 0.f ? 0.f : __expf(d);  // (NaN is not 0)
    float z = s.z * w, t = w == 0.f ? 0.f : w * (s.t + s.z * d);
    for (int o = 1; o < lanes; o <<= 1) {
        z += __shfl_xor_sync(0xffffffffu, z, o);
        t += __shfl_xor_sync(0xffffffffu, t, o);
    }
    return {m, z, t};
}

struct Shared {
    unsigned long long list[kWarps][kMaxTop];  // each warp's largest (a part's, in the cluster's join), descending
    unsigned long long largest[kMaxTop];       // the CTA's
    State warp_state[kWarps];
    State state;
    uint32_t group_max[32];
    float first_threshold;
    volatile float published[kWarps];
};

// The n largest of `lists` descending lists of kMaxTop keys (n of them used, the others 0), to
// out[0 .. n) in order.  Keys that are not 0 are unique, and 0 stands for nothing.
__device__ __forceinline__ void merge_lists(const unsigned long long (*list)[kMaxTop], int lists, int n,
                                            unsigned long long* out) {
    if ((int)threadIdx.x >= lists * n) return;  // (few keys: few warps)
    const int w = threadIdx.x / n, i = threadIdx.x - w * n;
    const unsigned long long mine = list[w][i];
    int before[kWarps];  // of list o, how many come before mine: a binary search, all lists at once
#pragma unroll
    for (int o = 0; o < kWarps; o++) before[o] = 0;
#pragma unroll
    for (int step = kMaxTop / 2; step > 0; step >>= 1) {
#pragma unroll
        for (int o = 0; o < kWarps; o++) {
            const unsigned long long k = list[o][before[o] + step - 1];
            if (k > mine || (k == mine && o < w)) before[o] += step;
        }
    }
    int rank = i;
#pragma unroll
    for (int o = 0; o < kWarps; o++) {
        const unsigned long long k = list[o][before[o]];  // the search ends one short of a whole list
        if (o != w && o < lists) rank += before[o] + (k > mine || (k == mine && o < w));
    }
    if (rank < n) out[rank] = mine;
}

__device__ __forceinline__ uint32_t mapa(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ unsigned long long ld_peer_u64(uint32_t addr) {
    unsigned long long v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr));
    return v;
}
__device__ __forceinline__ float ld_peer_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
    return v;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two f32 operations in one instruction.
__device__ __forceinline__ unsigned long long bits(const float2& a) { return reinterpret_cast<const unsigned long long&>(a); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<unsigned long long&>(d)) : "l"(bits(a)), "l"(bits(b)));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<unsigned long long&>(d)) : "l"(bits(a)), "l"(bits(b)));
    return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<unsigned long long&>(d)) : "l"(bits(a)), "l"(bits(b)), "l"(bits(c)));
    return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// The two elements of a word, in f32.
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
    if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w));
    else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

template <typename T>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) logprobs_kernel(const __grid_constant__ LogprobParams p, int parts) {
    constexpr int VEC = 16 / sizeof(T), U = kVecs, S = kStages, E = U * VEC, CHUNK = kThreads * E;
    constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
    // [S][U][kThreads] vectors, filled by the thread that sums them.  (128-byte aligned: copies to other places
    // took three times the shared-memory passes and twice the sectors from L2.)
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ Shared s;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.x / parts, part = blockIdx.x % parts, n = p.n_top;
    const T* x = static_cast<const T*>(p.logits) + (int64_t)row * p.row_stride;
    // 16-byte vectors of memory: vector v holds elements v * VEC - shift ..; the parts take
    // consecutive runs of whole chunks.  Every vector goes through the ring; what is outside the row is
    // -inf there, so that it has probability 0
    const int shift = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    const int64_t end = (int64_t)p.vocab + shift;
    const int chunks = (int)((end + CHUNK - 1) / CHUNK), inner0 = shift ? 1 : 0, inner1 = (int)(end / CHUNK);
    const int c0 = (int)((int64_t)chunks * part / parts), c1 = (int)((int64_t)chunks * (part + 1) / parts);

    constexpr uint32_t kSlot = U * kThreads * 16;  // bytes of a chunk
    const uint4* next = reinterpret_cast<const uint4*>(x - shift) + tid + (int64_t)c0 * (U * kThreads);  // to be loaded
    const uint32_t slots = smem_u32(ring) + tid * 16;
    uint32_t to_slot = 0, slot = 0;  // bytes into the ring: of the next load, of the chunk at hand
    const int whole0 = inner0, whole1 = min(inner1, c1);
    auto copy = [&](uint32_t dst, const uint4* src) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    };
    auto load = [&](int chunk) {  // chunks behind the last are not read
        const uint32_t dst = slots + to_slot;
        if (chunk >= whole0 && chunk < whole1) {
#pragma unroll
            for (int u = 0; u < U; u++) copy(dst + u * kThreads * 16, next + u * kThreads);
        } else if (chunk < c1) {  // an end of the row
#pragma unroll 1
            for (int u = 0; u < U; u++) {
                const int64_t e0 = (int64_t)chunk * CHUNK + (u * kThreads + tid) * VEC - shift;
                if (e0 >= 0 && e0 + VEC <= p.vocab) {
                    copy(dst + u * kThreads * 16, next + u * kThreads);
                    continue;
                }
                T* to = reinterpret_cast<T*>(ring + to_slot + (u * kThreads + tid) * 16);
                for (int i = 0; i < VEC; i++) to[i] = e0 + i >= 0 && e0 + i < p.vocab ? x[e0 + i] : static_cast<T>(-INFINITY);
            }
        }
        next += U * kThreads;
        to_slot = to_slot == (S - 1) * kSlot ? 0 : to_slot + kSlot;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // place in the row of element i of the E elements of thread t in a chunk
    auto place = [&](int chunk, int t, int i) {
        return (int64_t)chunk * CHUNK + (i / VEC) * (kThreads * VEC) + t * VEC + i % VEC - shift;
    };
#pragma unroll
    for (int i = 0; i < S - 1; i++) load(c0 + i);
    if (lane == 0) s.published[warp] = -INFINITY;

    State st = {-INFINITY, 0.f, 0.f};
    float c = 0.f, delta = 0.f, scale = 1.f;  // of st.m: m log2 e rounded, what was cut off, and 2^-delta
    unsigned long long mine = 0;               // lane i: the warp's i-th largest key
    // warps publish their k_share-th; the r_share-th largest of those bounds the n-th of all
    const int k_share = (n + 4) / 5, r_share = n > 0 ? (n + k_share - 1) / k_share : 1;
    float thr = -INFINITY;
    for (int chunk = c0; chunk < c1; chunk++) {
        asm volatile("cp.async.wait_group %0;" ::"n"(S - 2) : "memory");
        const uint32_t src = slots + slot;
        float mx = -INFINITY;
        uint32_t r[U * 4];
#pragma unroll
        for (int u = 0; u < U; u++)
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(r[4 * u]), "=r"(r[4 * u + 1]), "=r"(r[4 * u + 2]), "=r"(r[4 * u + 3])
                         : "r"(src + u * kThreads * 16)
                         : "memory");
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < E; i++) mx = fmaxf(mx, __uint_as_float(r[i]));
        } else {
            using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
            T2 top = reinterpret_cast<const T2&>(r[0]);
#pragma unroll
            for (int i = 1; i < E / 2; i++) top = __hmax2(top, reinterpret_cast<const T2&>(r[i]));
            const float2 f = unpack2<T>(reinterpret_cast<const uint32_t&>(top));
            mx = fmaxf(f.x, f.y);
        }
        auto pair = [&](int i) {  // elements i and i + 1, i even
            if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(r[i]), __uint_as_float(r[i + 1]));
            else return unpack2<T>(r[i / 2]);
        };
        load(chunk + S - 1);

        if (mx > st.m) {
            const float d = st.m - mx, w = __expf(d);
            st.t = w == 0.f ? 0.f : w * (st.t + st.z * d);
            st.z *= w;
            st.m = mx;
            c = mx * kLog2e;
            delta = fmaf(mx, kLog2e, -c);
            scale = ex2(-delta);
        }
        // y = (x - m) log2 e + delta in one multiply-add: delta is what rounding c cost
        bool plain = fabsf(st.m) < 1e6f;
        if (plain) {
            const float2 l2e = make_float2(kLog2e, kLog2e), off = make_float2(-c, -c);
            float2 z = make_float2(0.f, 0.f), t = make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < E; i += 2) {
                const float2 y = fma2(pair(i), l2e, off), e = make_float2(ex2(y.x), ex2(y.y));
                z = add2(z, e);
                t = fma2(e, y, t);
            }
            const float zs = z.x + z.y, ts = t.x + t.y;
            plain = ts == ts;  // 0 * -inf where a logit is -inf
            if (plain) {
                st.z += scale * zs;
                st.t += scale * kLn2 * (ts - delta * zs);
            }
        }
        if (!plain) {  // an end of the row, a logit of -inf or NaN, a huge maximum
            const float ref = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
            for (int i = 0; i < E; i += 2) {
                const float2 f = pair(i);
                const float d0 = max_nan(f.x - ref, -1000.f), d1 = max_nan(f.y - ref, -1000.f);  // e^-1000 is 0
                const float e0 = ex2(d0 * kLog2e), e1 = ex2(d1 * kLog2e);
                st.z += e0 + e1;
                st.t += e0 * d0 + e1 * d1;
            }
        }
        if (n > 0) {
            if (chunk == c0) {
                float g = mx;
#pragma unroll
                for (int o = 4; o > 0; o >>= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
                if ((tid & 7) == 0) s.group_max[tid >> 3] = ordered(g);
                __syncthreads();
                if (tid < 32) {
                    const uint32_t me = s.group_max[tid];
                    int rank = 0;
#pragma unroll
                    for (int i = 0; i < 32; i++) rank += s.group_max[i] > me || (s.group_max[i] == me && i < tid);
                    if (rank == n - 1) s.first_threshold = unordered(me);
                }
                __syncthreads();
                thr = s.first_threshold;
            }
            // lanes with an element to look at (a maximum skips NaN, which counts as largest here: the sum shows it)
            uint32_t look = __ballot_sync(0xffffffffu, !(mx < thr) || st.z != st.z);
            const bool found = look != 0;
            if (found) {
                __syncwarp();  // the other lanes' copies
                unsigned long long last = __shfl_sync(0xffffffffu, mine, n - 1);
                for (; look; look &= look - 1) {
                    const int t = warp * 32 + __ffs(look) - 1;
                    // lane i takes element i of that lane
                    const int64_t e = place(chunk, t, lane);
                    unsigned long long key = 0;
                    if (lane < E && e >= 0 && e < p.vocab) {
                        const float v = to_f32(*reinterpret_cast<const T*>(
                            ring + slot + lane / VEC * (kThreads * 16) + t * 16 + lane % VEC * sizeof(T)));
                        if (!(v < thr)) key = ((unsigned long long)ordered(v) << 32) | (uint32_t)~(uint32_t)e;
                    }
                    uint32_t todo = __ballot_sync(0xffffffffu, key > last);
                    while (todo) {
                        const int from = __ffs(todo) - 1;
                        const unsigned long long k = __shfl_sync(0xffffffffu, key, from);
                        const int at = __popc(__ballot_sync(0xffffffffu, mine > k));
                        const unsigned long long up = __shfl_up_sync(0xffffffffu, mine, 1);
                        if (lane >= at) mine = lane == at ? k : up;
                        last = __shfl_sync(0xffffffffu, mine, n - 1);
                        todo &= __ballot_sync(0xffffffffu, key > last) & ~(1u << from);
                    }
                }
                if (last) thr = fmaxf(thr, unordered((uint32_t)(last >> 32)));
                const unsigned long long share = __shfl_sync(0xffffffffu, mine, k_share - 1);
                if (lane == 0 && share) {
                    const float f = unordered((uint32_t)(share >> 32));
                    s.published[warp] = f == f ? f : INFINITY;  // (NaN counts as largest)
                }
            }
            if (found || chunk % 4 == 0) {
                const float v = s.published[lane % kWarps];
                int rank = 0;
#pragma unroll
                for (int o = 1; o < kWarps; o++) {
                    const float u = __shfl_xor_sync(0xffffffffu, v, o);
                    rank += u > v || (u == v && (lane ^ o) < lane);
                }
                const float shared = __shfl_sync(0xffffffffu, v, __ffs(__ballot_sync(0xffffffffu, rank == r_share - 1)) - 1);
                thr = fmaxf(thr, shared);
            }
        }
        slot = slot == (S - 1) * kSlot ? 0 : slot + kSlot;
    }

    // the CTA's state and list
    st = join_lanes(st, 32);
    if (lane == 0) s.warp_state[warp] = st;
    s.list[warp][lane] = lane < n ? mine : 0;
    __syncthreads();
    merge_lists(s.list, kWarps, n, s.largest);
    if (warp == 0) {
        st = join_lanes(s.warp_state[lane % kWarps], kWarps);
        if (lane == 0) s.state = st;
    }
    if (parts > 1) {
        cluster_sync();  // every part's state and list are complete
        if (part == 0) {
            if (warp < parts) s.list[warp][lane] = lane < n ? ld_peer_u64(mapa(smem_u32(&s.largest[lane]), warp)) : 0;
            if (warp == 0) {
                const int q = lane & (parts - 1);
                st = {ld_peer_f32(mapa(smem_u32(&s.state.m), q)), ld_peer_f32(mapa(smem_u32(&s.state.z), q)),
                      ld_peer_f32(mapa(smem_u32(&s.state.t), q))};
                st = join_lanes(st, parts);
            }
        }
        cluster_sync();  // nobody leaves, or is overwritten, while its shared memory is read
        if (part != 0) return;
        if (tid == 0) s.state = st;
        merge_lists(s.list, parts, n, s.largest);
    }
    __syncthreads();
    const State all = s.state;
    const float log_z = logf(all.z);
    if (tid < n) {
        const unsigned long long k = s.largest[tid];
        p.top_id[(int64_t)row * n + tid] = (int32_t) ~(uint32_t)k;
        p.top_logprob[(int64_t)row * n + tid] = (unordered((uint32_t)(k >> 32)) - all.m) - log_z;
    }
    if (tid == 0) {
        if (p.logprob) {
            const int id = p.token[row];
            p.logprob[row] = id >= 0 && id < p.vocab ? (to_f32(x[id]) - all.m) - log_z : __int_as_float(0x7fc00000);
        }
        if (p.entropy) p.entropy[row] = log_z - all.t / all.z;
    }
}

template <typename T>
cudaError_t launch_t(const LogprobParams& p, int parts, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((int64_t)p.rows * parts));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kRing;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = parts;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = parts > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, logprobs_kernel<T>, p, parts);
}

}  // namespace

cudaError_t logprobs_init_device() {
    cudaError_t e = cudaFuncSetAttribute(logprobs_kernel<float>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRing);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(logprobs_kernel<__half>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRing);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(logprobs_kernel<__nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRing);
    return e;
}

cudaError_t launch_logprobs(int type, const LogprobParams& p, int sms, cudaStream_t st) {
    // CTAs per row: up to two for each SM in all, while each still has two chunks (148 bf16 rows of 128256 in
    // two parts 19 us, 149 in one 22, 300 in one 29; two parts for 1500 rows 115 instead of 88)
    const int chunk = kThreads * kVecs * (type == TPTC_TYPE_F32 ? 4 : 8);
    int parts = 1;
    while (parts < kMaxParts && (int64_t)p.rows * parts * 2 <= 2 * sms && p.vocab / (parts * 2) >= 2 * chunk) parts *= 2;
    if (type == TPTC_TYPE_F16) return launch_t<__half>(p, parts, st);
    if (type == TPTC_TYPE_BF16) return launch_t<__nv_bfloat16>(p, parts, st);
    return launch_t<float>(p, parts, st);
}

}  // namespace tptc
