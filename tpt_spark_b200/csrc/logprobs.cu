// logprobs.cu -- log probabilities of given tokens, entropy and the largest alternatives of each
// row of logits, in one pass over the logits.
//
// With m = max x, z = sum e^(x - m) and t = sum e^(x - m) (x - m):
//     log p(i) = x_i - m - log z,      entropy = log z - t / z.
// A thread keeps (m, z, t) of its elements and moves them to a new maximum m' by
// z <- z a, t <- a (t + z (m - m')), a = e^(m - m'); the CTA's states join in thread order.
//
// The n largest, exactly and with ties by lowest index: an element that beats the running
// threshold goes to a shared buffer as one 64-bit key (ordered value bits, then ~index), which
// makes keys unique and their order the wanted one.  The first threshold is the n-th largest of
// 32 group maxima of the first chunk (n elements are at least that large); the buffer is
// cut back to its n largest, which raises the threshold, when it fills.  After the first chunk
// only about n ln(vocab / chunk) elements pass.
//
// One CTA per row streams the logits (HBM bound); with few rows a cluster of 2, 4 or 8 CTAs
// shares one row and joins through distributed shared memory (latency bound).
#include <algorithm>

#include "serve.h"

namespace tptc {

namespace {

constexpr int kThreads = 256;
constexpr int kElems = 16;                   // elements per thread and chunk
constexpr int kChunk = kThreads * kElems;
constexpr int kLimit = 512;                  // buffered keys before they are cut back
constexpr int kCap = kLimit + kChunk;        // a chunk can push every element

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
// The state of two disjoint sets; an empty set has m = -inf, z = t = 0.
__device__ __forceinline__ State join(const State& a, const State& b) {
    const float m = fmaxf(a.m, b.m);
    State r = {m, 0.f, 0.f};
    const State* both[2] = {&a, &b};
#pragma unroll
    for (int i = 0; i < 2; i++) {
        if (both[i]->z == 0.f) continue;  // nothing with a probability (NaN is not 0)
        const float d = both[i]->m - m, w = __expf(d);
        r.z += both[i]->z * w;
        r.t += w == 0.f ? 0.f : w * (both[i]->t + both[i]->z * d);
    }
    return r;
}

struct Shared {
    unsigned long long key[kCap];
    unsigned long long kept[2 * kLimit];
    unsigned long long group[32];
    unsigned long long bound;
    State warp_state[kThreads / 32];
    uint32_t group_max[32];
    State state;
    float threshold;
    int count, n_kept;
};

// Cuts key[0 .. count) back to its n largest, in descending order in key[0 ..); returns how
// many there are.  Every thread of the CTA calls it; key is complete.
__device__ int keep_largest(Shared& s, int count, int n) {
    const int tid = threadIdx.x;
    unsigned long long* list = s.key;
    if (count > 64) {
        // n of the 32 group maxima are at least the n-th of them: what is below is out
        unsigned long long best = 0;
        for (int i = tid; i < count; i += kThreads) best = max(best, s.key[i]);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        if ((tid & 7) == 0) s.group[tid >> 3] = best;
        if (tid == 0) s.n_kept = 0;
        __syncthreads();
        if (tid < 32) {
            const unsigned long long mine = s.group[tid];
            int rank = 0;
            for (int i = 0; i < 32; i++) rank += s.group[i] > mine || (s.group[i] == mine && i < tid);
            if (rank == n - 1) s.bound = mine;
        }
        __syncthreads();
        const unsigned long long bound = s.bound;
        for (int i = tid; i < count; i += kThreads)
            if (s.key[i] >= bound) {
                const int at = atomicAdd(&s.n_kept, 1);
                if (at < 2 * kLimit) s.kept[at] = s.key[i];
            }
        __syncthreads();
        if (s.n_kept <= 2 * kLimit) {
            list = s.kept;
            count = s.n_kept;
        }
    }
    // ranks by counting (keys are unique); the largest n move to their places
    if (list == s.key) {
        constexpr int PER = (kCap + kThreads - 1) / kThreads;
        unsigned long long mine[PER];
        int rank[PER], k = 0;
        for (int i = tid; i < count; i += kThreads, k++) {
            mine[k] = s.key[i];
            rank[k] = 0;
            for (int j = 0; j < count; j++) rank[k] += s.key[j] > mine[k];
        }
        __syncthreads();
        for (int i = 0; i < k; i++)
            if (rank[i] < n) s.key[rank[i]] = mine[i];
    } else {
        for (int i = tid; i < count; i += kThreads) {
            const unsigned long long mine = list[i];
            int rank = 0;
            for (int j = 0; j < count; j++) rank += list[j] > mine;
            if (rank < n) s.key[rank] = mine;
        }
    }
    __syncthreads();
    return min(count, n);
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
__device__ __forceinline__ int ld_peer_s32(uint32_t addr) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr));
    return v;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_kernel(const __grid_constant__ LogprobParams p, int parts) {
    constexpr int VEC = 16 / sizeof(T), U = kElems / VEC;
    extern __shared__ __align__(16) uint8_t smem[];
    Shared& s = *reinterpret_cast<Shared*>(smem);
    const int tid = threadIdx.x, row = blockIdx.x / parts, part = blockIdx.x % parts, n = p.n_top;
    const T* x = static_cast<const T*>(p.logits) + (int64_t)row * p.row_stride;
    // 16-byte vectors of memory: vector v holds elements v * VEC - shift ..; the parts take
    // consecutive runs of whole chunks
    const int shift = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    const int64_t n_vec = ((int64_t)p.vocab + shift + VEC - 1) / VEC;
    const int64_t chunks = (n_vec + kThreads * U - 1) / (kThreads * U);
    const int64_t c0 = chunks * part / parts, c1 = chunks * (part + 1) / parts;

    if (tid == 0) s.count = 0;
    __syncthreads();

    auto load = [&](int64_t chunk, float (&v)[kElems]) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t vec = (chunk * U + u) * kThreads + tid, e0 = vec * VEC - shift;
            if (e0 >= 0 && e0 + VEC <= p.vocab) {
                const uint4 w = __ldcs(reinterpret_cast<const uint4*>(x + e0));
                const uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if constexpr (sizeof(T) == 4) {
                        v[u * VEC + i] = __uint_as_float(r[i]);
                    } else {
                        const T* h = reinterpret_cast<const T*>(&r[i]);
                        v[u * VEC + 2 * i] = to_f32(h[0]);
                        v[u * VEC + 2 * i + 1] = to_f32(h[1]);
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < VEC; i++) {
                    const int64_t e = e0 + i;
                    v[u * VEC + i] = e >= 0 && e < p.vocab ? to_f32(x[e]) : -INFINITY;
                }
            }
        }
    };

    State st = {-INFINITY, 0.f, 0.f};
    float thr = -INFINITY;
    float cur[kElems], nxt[kElems];
    if (c0 < c1) load(c0, cur);
    for (int64_t chunk = c0; chunk < c1; chunk++) {
        if (chunk + 1 < c1) load(chunk + 1, nxt);
        float mx = cur[0];
#pragma unroll
        for (int i = 1; i < kElems; i++) mx = fmaxf(mx, cur[i]);
        if (mx > st.m) {
            const float d = st.m - mx, w = __expf(d);
            st.t = w == 0.f ? 0.f : w * (st.t + st.z * d);
            st.z *= w;
            st.m = mx;
        }
        const float ref = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
        for (int i = 0; i < kElems; i++) {
            const float d = cur[i] - ref, e = __expf(d);
            st.z += e;
            st.t += e * fmaxf(d, -1000.f);  // e is 0 there; -inf would make 0 * inf
        }
        if (n > 0) {
            const bool first = chunk == c0;
            if (first) {  // the n-th largest of the maxima of 32 groups of 8 threads
                float g = mx;
#pragma unroll
                for (int o = 4; o > 0; o >>= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
                if ((tid & 7) == 0) s.group_max[tid >> 3] = ordered(g);
                __syncthreads();
                if (tid < 32) {
                    const uint32_t mine = s.group_max[tid];
                    int rank = 0;
                    for (int i = 0; i < 32; i++) rank += s.group_max[i] > mine || (s.group_max[i] == mine && i < tid);
                    if (rank == n - 1) s.threshold = unordered(mine);
                }
                __syncthreads();
                thr = s.threshold;
            }
            bool full = false;
#pragma unroll
            for (int i = 0; i < kElems; i++) {
                // later chunks hold higher indices only: an equal element loses there
                if (first ? !(cur[i] < thr) : !(cur[i] <= thr)) {
                    const int u = i / VEC;
                    const int64_t e = ((chunk * U + u) * kThreads + tid) * VEC - shift + i % VEC;
                    if (e >= 0 && e < p.vocab) {
                        const int at = atomicAdd(&s.count, 1);
                        s.key[at] = ((unsigned long long)ordered(cur[i]) << 32) | (uint32_t)~(uint32_t)e;
                        full |= at >= kLimit;
                    }
                }
            }
            if (__syncthreads_or(full)) {
                const int kept = keep_largest(s, s.count, n);
                if (tid == 0) s.count = kept;
                if (kept == n) thr = unordered((uint32_t)(s.key[n - 1] >> 32));
                __syncthreads();
            }
        }
#pragma unroll
        for (int i = 0; i < kElems; i++) cur[i] = nxt[i];
    }

    // the CTA's state, in a fixed order
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const State other = {__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.z, o),
                             __shfl_xor_sync(0xffffffffu, st.t, o)};
        st = (tid & o) ? join(other, st) : join(st, other);
    }
    if ((tid & 31) == 0) s.warp_state[tid >> 5] = st;
    __syncthreads();
    int count = s.count;
    if (n > 0) count = keep_largest(s, count, n);
    if (tid == 0) {
        st = s.warp_state[0];
        for (int w = 1; w < kThreads / 32; w++) st = join(st, s.warp_state[w]);
        s.state = st;
        s.count = count;
    }
    if (parts > 1) {
        cluster_sync();  // every part's state and list are complete
        if (part == 0) {
            // the other parts' lists behind this one's, then the n largest of all
            int total = count;
            for (int q = 1; q < parts; q++) {
                const int c = n > 0 ? ld_peer_s32(mapa(smem_u32(&s.count), q)) : 0;
                if (tid < c) s.key[total + tid] = ld_peer_u64(mapa(smem_u32(&s.key[tid]), q));
                total += c;
            }
            if (tid == 0) {
                for (int q = 1; q < parts; q++) {
                    const State other = {ld_peer_f32(mapa(smem_u32(&s.state.m), q)),
                                         ld_peer_f32(mapa(smem_u32(&s.state.z), q)),
                                         ld_peer_f32(mapa(smem_u32(&s.state.t), q))};
                    st = join(st, other);
                }
                s.state = st;
            }
            __syncthreads();
            if (n > 0) count = keep_largest(s, total, n);
        }
        cluster_sync();  // nobody leaves while its shared memory is read
        if (part != 0) return;
    } else {
        __syncthreads();
    }
    const State all = s.state;
    const float log_z = logf(all.z);
    if (tid < n) {
        const unsigned long long k = s.key[tid];
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
    cfg.dynamicSmemBytes = sizeof(Shared);
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
    cudaError_t e = cudaFuncSetAttribute(logprobs_kernel<float>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Shared));
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(logprobs_kernel<__half>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Shared));
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(logprobs_kernel<__nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Shared));
    return e;
}

cudaError_t launch_logprobs(int type, const LogprobParams& p, int sms, cudaStream_t st) {
    // CTAs per row: as many as fit the GPU twice over, while each still has two chunks
    int parts = 1;
    while (parts < 8 && (int64_t)p.rows * parts * 2 <= 2 * sms && p.vocab / (parts * 2) >= 2 * kChunk) parts *= 2;
    if (type == TPTC_TYPE_F16) return launch_t<__half>(p, parts, st);
    if (type == TPTC_TYPE_BF16) return launch_t<__nv_bfloat16>(p, parts, st);
    return launch_t<float>(p, parts, st);
}

}  // namespace tptc
