// kv8.cu -- the paged 8-bit KV cache: appending a ragged batch of new keys and values (with the
// position rotation of q and k in the same pass) and reading positions back as dense rows.
//
// Append.  A page of one kv head has one scale s, and its codes are c = rint(x / s), |c| <= 127.
// With a = max |x| over the page's new rows, s' = max(s, a / 127); where s' > s the earlier codes
// become rint(c s / s'), so a value moves by at most half a step s' each time the scale grows.
// The maximum over the page couples all of its new rows, hence the split: one CTA per (sequence,
// touched page, kv head), which keeps the page's rotated rows in registers between the maximum
// and the rounding (each input is read once).  A second CTA beside it rotates the query rows of
// its head group and positions, four heads of a token per thread with one pair of cos and sin vectors, so one launch moves q, k and
// v.  Bound by HBM for prompts and by launch latency for
// decode steps: 44 us for 7900 bf16 tokens of 32 heads on 8 (194 MB, 4.4 TB/s), 6.3 us for one token of each of 64 sequences.
#include <algorithm>

#include "serve.h"

namespace tptc {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ void flag(int32_t* status) {
    if (status) atomicExch(status, TPTC_ERR_ARG);
}

// The rows of sequence b (from packed row lo, position begin): how many, or -1 where they are out of range.
__device__ __forceinline__ int rows_of(const tptc_kv8& c, const int32_t* cu, const int32_t* start, int n_rows, int most,
                                       int rope_rows, int b, int& lo, int& begin) {
    lo = cu[b];
    begin = start[b];
    const int hi = cu[b + 1];
    if (lo == hi) return 0;
    const int64_t cap = c.max_pages * c.page, end = (int64_t)begin + hi - lo;
    const bool in = lo >= 0 && hi > lo && hi <= n_rows && hi - lo <= most && begin >= 0 && end <= cap &&
                    (rope_rows < 0 || end <= rope_rows);
    return in ? hi - lo : -1;
}

// A CTA's work: the rows of sequence b that lie in one page (page u of those that it touches).
struct Span {
    int first, n;   // packed row of the first, and how many
    int off;        // their first row in the page
    int pos;        // position of the first
    int64_t entry;  // of the page table
};
// The k-th page that any sequence touches, in order, as (sequence, its page); -1 behind the last.  (A call: it is
// over before the rows' registers are in use.)
__device__ __noinline__ int2 counted_unit(const tptc_kv8& c, const int32_t* cu, const int32_t* start, int n_rows, int most,
                                          int rope_rows, int k) {
    __shared__ int s_sum[kThreads / 32], s_at[2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, shift = 31 - __clz(c.page);
    int before = 0;
    for (int b0 = 0; b0 < c.n_seq; b0 += kThreads) {
        const int b = b0 + threadIdx.x;
        int lo, begin;
        const int n = b < c.n_seq ? rows_of(c, cu, start, n_rows, most, rope_rows, b, lo, begin) : 0;
        if (n < 0 && blockIdx.x == 0) flag(c.status);
        const int t = n > 0 ? ((begin + n - 1) >> shift) - (begin >> shift) + 1 : 0;
        int incl = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) s_sum[warp] = incl;
        __syncthreads();
        int lead = before;
        for (int w = 0; w < kThreads / 32; w++) {
            if (w < warp) lead += s_sum[w];
            before += s_sum[w];
        }
        lead += incl - t;
        if (lead <= k && k < lead + t) s_at[0] = b, s_at[1] = k - lead;
        __syncthreads();
        if (k < before && blockIdx.x != 0) break;  // (the first CTA sees all, and reports)
    }
    return k < before ? make_int2(s_at[0], s_at[1]) : make_int2(-1, 0);
}

// units > 0: unit k is page k % units of sequence k / units.  units 0: units are counted (a batch whose longest
// sequence is far from the others: 63 sequences of one row beside one of 8192 took 289 us in the first form, 59 in
// this one).
__device__ __forceinline__ bool page_span(const tptc_kv8& c, const int32_t* cu, const int32_t* start, int n_rows,
                                          int most, int rope_rows, int units, int k, Span& s) {
    const int shift = 31 - __clz(c.page);
    int b, u, lo, begin;
    if (units > 0) {
        b = k / units;
        u = k - b * units;
    } else {
        const int2 at = counted_unit(c, cu, start, n_rows, most, rope_rows, k);
        if (at.x < 0) return false;
        b = at.x;
        u = at.y;
    }
    const int n = rows_of(c, cu, start, n_rows, most, rope_rows, b, lo, begin);
    if (n < 0 && u == 0 && threadIdx.x == 0) flag(c.status);
    const int p = (begin >> shift) + u, r0 = max(begin, p << shift), r1 = min(begin + n, (p << shift) + c.page);
    if (n <= 0 || p > (begin + n - 1) >> shift) return false;
    s.first = lo - begin + r0;
    s.n = r1 - r0;
    s.off = r0 & (c.page - 1);
    s.pos = r0;
    s.entry = (int64_t)b * c.max_pages + p;
    return true;
}

// A page id as it is (id), and whether it is in the cache; one that is not is flagged and not followed.
__device__ __forceinline__ bool in_cache(const tptc_kv8& c, int id) {
    const bool in = id >= 0 && id < c.n_pages;
    if (!in && threadIdx.x == 0) flag(c.status);
    return in;
}

// The cos and sin that the eight elements of lane lg of a row at `pos` take (pairs: four of each).
struct Angles {
    float c[8], s[8];
};
__device__ __forceinline__ void load_angles(const tptc_rope& r, int lg, int pos, bool in, Angles& a) {
    const int e = 8 * lg, half = r.dim / 2;
    if (!in || e >= r.dim) return;
    const int64_t at = (int64_t)pos * half + (r.halves ? (e >= half ? e - half : e) : e / 2);
    const float4* c = reinterpret_cast<const float4*>(r.cos + at);
    const float4* s = reinterpret_cast<const float4*>(r.sin + at);
    reinterpret_cast<float4*>(a.c)[0] = __ldg(c);
    reinterpret_cast<float4*>(a.s)[0] = __ldg(s);
    if (r.halves) {
        reinterpret_cast<float4*>(a.c)[1] = __ldg(c + 1);
        reinterpret_cast<float4*>(a.s)[1] = __ldg(s + 1);
    }
}

// The eight elements of lane lg of a row (held by a group of lanes), rotated.  Each product and sum is
// rounded by itself, as the framework's other rotations do.  Every lane of the warp takes part (the
// halves form exchanges vectors as they were loaded; for the first half the partner's sign turns with them).
template <typename T>
__device__ __forceinline__ void rotate8(const Raw8<T>& w, float (&x)[8], int lg, const tptc_rope& r, const Angles& a) {
    unpack8<T>(w, x);
    const int e = 8 * lg;
    if (!r.halves) {
        if (e >= r.dim) return;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float u = x[2 * i], v = x[2 * i + 1];
            x[2 * i] = __fsub_rn(__fmul_rn(u, a.c[i]), __fmul_rn(v, a.s[i]));
            x[2 * i + 1] = __fadd_rn(__fmul_rn(u, a.s[i]), __fmul_rn(v, a.c[i]));
        }
        return;
    }
    const int half = r.dim / 2, delta = half / 8, lane = threadIdx.x & 31;
    const int src = e >= r.dim ? lane : e >= half ? lane - delta : lane + delta;
    const uint32_t sign = e >= half ? 0u : sizeof(T) == 4 ? 0x80000000u : 0x80008000u;
    const uint32_t* wi = reinterpret_cast<const uint32_t*>(&w);
    Raw8<T> o;
    uint32_t* wo = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
    for (int i = 0; i < 2 * (int)sizeof(T); i++) wo[i] = __shfl_sync(0xffffffffu, wi[i], src) ^ sign;
    if (e >= r.dim) return;
    float y[8];
    unpack8<T>(o, y);
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = __fadd_rn(__fmul_rn(x[i], a.c[i]), __fmul_rn(y[i], a.s[i]));
}

// Scale of a page after values of magnitude up to `top` joined it (inf or NaN: not finite).
__device__ __forceinline__ float grown_scale(float old, float top) {
    if (!(top <= 3.402823466e38f) || isnan(old)) return __int_as_float(0x7fc00000);
    const float s = fmaxf(old, __fmul_rn(top, 1.f / 127.f));
    return s < 1.17549435e-38f ? 0.f : s;
}

__device__ __forceinline__ int code_of(float x, float inv) {
    // a NaN (only where the scale is NaN) converts to 0
    return max(-127, min(127, __float2int_rn(__fmul_rn(x, inv))));
}

__device__ __forceinline__ void store_codes(int8_t* dst, const float (&x)[8], float inv) {
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        w[h] = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) w[h] |= (uint32_t)(code_of(x[4 * h + i], inv) & 255) << (8 * i);
    }
    *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
}

// The earlier codes of the page (n of them, a multiple of 16) after the scale grew.
__device__ __forceinline__ void rescale_codes(int8_t* codes, int n, float ratio) {
    for (int i = threadIdx.x; i < n / 16; i += kThreads) {
        uint4* at = reinterpret_cast<uint4*>(codes) + i;
        uint4 w = *at;
        uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            uint32_t o = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int c = (int8_t)(r[k] >> (8 * j));
                o |= (uint32_t)(__float2int_rn(__fmul_rn((float)c, ratio)) & 255) << (8 * j);
            }
            r[k] = o;
        }
        *at = make_uint4(r[0], r[1], r[2], r[3]);
    }
}

// NR: passes of the CTA over a page's rows (16 or 32 rows each).
template <typename T, int HD, int NR>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 ? 2 : NR == 4 ? 3 : 4)
    kv8_append_kernel(const __grid_constant__ Kv8Append p) {
    constexpr int GS = HD == 64 ? 8 : 16;  // lanes per row (12 of 16 work at head_dim 96)
    constexpr int RP = kThreads / GS;
    __shared__ float s_top[2][kThreads / 32];
    const int tid = threadIdx.x, lg = tid % GS, grp = tid / GS, c = 8 * lg;
    const bool lane_in = c < HD;
    const int roles = p.q_out ? 2 : 1, role = blockIdx.x % roles, rest = blockIdx.x / roles;
    const int h = rest % p.c.n_kv;
    Span s;
    if (!page_span(p.c, p.cu, p.start, p.n_tokens, p.max_new, p.rope.dim ? p.rope.rows : -1, p.units, rest / p.c.n_kv, s)) return;

    if (role == 1) {  // the queries of this head group at the same positions: up to B heads of a token at a time
        constexpr int B = 4;
        const int G = p.n_heads / p.c.n_kv, sets = (G + B - 1) / B, items = s.n * sets;
        const T* qin = static_cast<const T*>(p.q) + (int64_t)s.first * p.q_stride + (int64_t)h * G * HD + c;
        T* qout = static_cast<T*>(p.q_out) + ((int64_t)s.first * p.n_heads + (int64_t)h * G) * HD + c;
        for (int w0 = 0; w0 < items; w0 += RP) {
            const int w = w0 + grp, t = sets == 1 ? w : w / sets, g0 = sets == 1 ? 0 : (w - t * sets) * B;
            const int n = lane_in && w < items ? min(B, G - g0) : 0;
            const T* src = qin + (int64_t)t * p.q_stride + g0 * HD;
            T* dst = qout + ((int64_t)t * p.n_heads + g0) * HD;
            Raw8<T> v[B];
            Angles a;
#pragma unroll
            for (int i = 0; i < B; i++)
                if (i < n) v[i] = load_raw8(src + i * HD);
            if (p.rope.dim) load_angles(p.rope, lg, s.pos + t, n > 0, a);
#pragma unroll
            for (int i = 0; i < B; i++) {
                float x[8];
                if (p.rope.dim) rotate8<T>(v[i], x, lg, p.rope, a);
                else unpack8<T>(v[i], x);
                if (i < n) store8(dst + i * HD, x);
            }
        }
        return;
    }
    const int page_id = p.c.table[s.entry];  // (looked at after the rows are on their way)
    const T* kin = static_cast<const T*>(p.k) + (int64_t)s.first * p.k_stride + h * HD + c;
    const T* vin = static_cast<const T*>(p.v) + (int64_t)s.first * p.v_stride + h * HD + c;
    float xk[NR][8], xv[NR][8];
    float top_k = 0.f, top_v = 0.f;
    bool odd_k = false, odd_v = false;  // a value that is not finite
    {
        Raw8<T> wk[NR], wv[NR];
#pragma unroll
        for (int i = 0; i < NR; i++) {
            const int row = grp + i * RP;
            wk[i] = wv[i] = Raw8<T>{};
            if (lane_in && row < s.n) {
                wk[i] = load_raw8(kin + row * p.k_stride);
                wv[i] = load_raw8(vin + row * p.v_stride);
            }
        }
#pragma unroll
        for (int i = 0; i < NR; i++) {
            const int row = grp + i * RP;
            Angles a;
            if (p.rope.dim) {
                const bool in = lane_in && row < s.n;
                load_angles(p.rope, lg, s.pos + row, in, a);
                rotate8<T>(wk[i], xk[i], lg, p.rope, a);
                if (!in)  // (angles that were not loaded)
#pragma unroll
                    for (int e = 0; e < 8; e++) xk[i][e] = 0.f;
            } else {
                unpack8<T>(wk[i], xk[i]);
            }
            unpack8<T>(wv[i], xv[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < NR; i++) {
        const int row = grp + i * RP;
        const bool in = lane_in && row < s.n;
        if (in && p.k_out)
            store8(static_cast<T*>(p.k_out) + ((int64_t)(s.first + row) * p.c.n_kv + h) * HD + c, xk[i]);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float a = fabsf(xk[i][e]), d = fabsf(xv[i][e]);
            odd_k |= !(a <= 3.402823466e38f);
            odd_v |= !(d <= 3.402823466e38f);
            top_k = fmaxf(top_k, a);
            top_v = fmaxf(top_v, d);
        }
    }
    if (odd_k) top_k = INFINITY;
    if (odd_v) top_v = INFINITY;
    top_k = warp_max(top_k);
    top_v = warp_max(top_v);
    if ((tid & 31) == 0) s_top[0][tid >> 5] = top_k, s_top[1][tid >> 5] = top_v;

    const bool store = in_cache(p.c, page_id);
    const int64_t at = (int64_t)page_id * p.c.n_kv + h;
    float old_k = 0.f, old_v = 0.f;
    if (store && s.off > 0) old_k = p.c.k_scale[at], old_v = p.c.v_scale[at];

    __syncthreads();  // the maxima are in; every thread has read the old scales
    if (!store) return;
    top_k = s_top[0][0], top_v = s_top[1][0];
#pragma unroll
    for (int w = 1; w < kThreads / 32; w++) top_k = fmaxf(top_k, s_top[0][w]), top_v = fmaxf(top_v, s_top[1][w]);
    const float new_k = grown_scale(old_k, top_k), new_v = grown_scale(old_v, top_v);
    int8_t* ck = p.c.k + at * p.c.page * HD;
    int8_t* cv = p.c.v + at * p.c.page * HD;
    const float inv_k = new_k > 0.f ? __frcp_rn(new_k) : 0.f, inv_v = new_v > 0.f ? __frcp_rn(new_v) : 0.f;
#pragma unroll
    for (int i = 0; i < NR; i++) {
        const int row = grp + i * RP;
        if (!lane_in || row >= s.n) continue;
        store_codes(ck + (s.off + row) * HD + c, xk[i], inv_k);
        store_codes(cv + (s.off + row) * HD + c, xv[i], inv_v);
    }
    if (s.off > 0) {  // (a scale that is NaN compares false: the codes stay)
        if (new_k > old_k) rescale_codes(ck, s.off * HD, __fdiv_rn(old_k, new_k));
        if (new_v > old_v) rescale_codes(cv, s.off * HD, __fdiv_rn(old_v, new_v));
    }
    if (tid == 0) p.c.k_scale[at] = new_k, p.c.v_scale[at] = new_v;
}

// Sixteen codes as values: byte b of a word, offset to 0..255, in the mantissa of 2^23 + b, is exact.
template <typename T>
__device__ __forceinline__ void store_values(T* dst, const uint4& w, float scale) {
    const uint32_t r[4] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u, w.z ^ 0x80808080u, w.w ^ 0x80808080u};
    float x[2][8];
#pragma unroll
    for (int k = 0; k < 4; k++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float f = __uint_as_float(__byte_perm(r[k], 0x4b000000u, 0x7440 + j)) - 8388736.f;
            x[k >> 1][(k & 1) * 4 + j] = __fmul_rn(f, scale);
        }
    store8(dst, x[0]);
    store8(dst + 8, x[1]);
}

// One CTA per (sequence, page, group of kv heads): 16 codes per load, kReadLoads of K and of V in flight per
// thread; a page's rows of one head are contiguous, so that loads and stores both run along head_dim.  HBM bound:
// 27 us for 21k positions of 8 heads of 128 (130 MB, 4.8 TB/s; 5.8 TB/s for ten times that), 3.5 us for 300.
constexpr int kReadLoads = 2;  // (and 5 CTAs per SM: 255 us for 240k positions, 298 with 4 loads and 3 CTAs)
template <typename T, int HD, bool COUNTED>  // (both forms in one kernel: 29.4 us for 27.1)
__global__ void __launch_bounds__(kThreads, 5) kv8_read_kernel(const __grid_constant__ Kv8Read p) {
    constexpr int CH = HD / 16;
    const int groups = (p.c.n_kv + p.heads_per_cta - 1) / p.heads_per_cta;
    const int g = blockIdx.x % groups;
    Span s;
    if (!page_span(p.c, p.cu, p.start, p.n_tokens, p.max_rows, -1, COUNTED ? 0 : max(p.units, 1), blockIdx.x / groups, s)) return;
    const int page_id = p.c.table[s.entry];
    if (!in_cache(p.c, page_id)) return;
    const int h0 = g * p.heads_per_cta, heads = min(p.heads_per_cta, p.c.n_kv - h0);
    const int64_t at = (int64_t)page_id * p.c.n_kv + h0;
    const int8_t *k = p.c.k + at * p.c.page * HD, *v = p.c.v + at * p.c.page * HD;
    const int shift = 31 - __clz(p.c.page), total = heads * p.c.page * CH;
    for (int i0 = 0; i0 < total; i0 += kReadLoads * kThreads) {
        uint4 wk[kReadLoads], wv[kReadLoads];
        float sk[kReadLoads], sv[kReadLoads];
        int64_t dst[kReadLoads];
#pragma unroll
        for (int e = 0; e < kReadLoads; e++) {
            const int i = i0 + e * kThreads + threadIdx.x, r = i / CH, hh = r >> shift, row = (r & (p.c.page - 1)) - s.off;
            dst[e] = i < total && row >= 0 && row < s.n
                         ? ((int64_t)(s.first + row) * p.c.n_kv + h0 + hh) * HD + (i - r * CH) * 16
                         : -1;
            if (dst[e] < 0) continue;
            if (p.k_out) wk[e] = __ldcs(reinterpret_cast<const uint4*>(k) + i), sk[e] = p.c.k_scale[at + hh];
            if (p.v_out) wv[e] = __ldcs(reinterpret_cast<const uint4*>(v) + i), sv[e] = p.c.v_scale[at + hh];
        }
#pragma unroll
        for (int e = 0; e < kReadLoads; e++) {
            if (dst[e] < 0) continue;
            if (p.k_out) store_values(static_cast<T*>(p.k_out) + dst[e], wk[e], sk[e]);
            if (p.v_out) store_values(static_cast<T*>(p.v_out) + dst[e], wv[e], sv[e]);
        }
    }
}

template <typename P>
cudaError_t launch(void (*kernel)(P), int64_t ctas, const P& p, cudaStream_t st) {
    if (ctas <= 0 || ctas > 0x7fffffff) return cudaErrorInvalidConfiguration;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = st;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <typename T, int HD>
cudaError_t append_hd(const Kv8Append& p, int64_t ctas, cudaStream_t st) {
    constexpr int RP = kThreads / (HD == 64 ? 8 : 16);
    const int passes = (p.c.page + RP - 1) / RP;
    if (passes <= 1) return launch(kv8_append_kernel<T, HD, 1>, ctas, p, st);
    if (passes == 2) return launch(kv8_append_kernel<T, HD, 2>, ctas, p, st);
    if constexpr (HD != 64) return launch(kv8_append_kernel<T, HD, 4>, ctas, p, st);
    return cudaErrorInvalidValue;
}

template <typename T>
cudaError_t append_t(const Kv8Append& p, int64_t ctas, cudaStream_t st) {
    if (p.c.head_dim == 64) return append_hd<T, 64>(p, ctas, st);
    if (p.c.head_dim == 96) return append_hd<T, 96>(p, ctas, st);
    return append_hd<T, 128>(p, ctas, st);
}

template <typename T, int HD>
cudaError_t read_hd(const Kv8Read& p, int64_t ctas, cudaStream_t st) {
    if (p.units > 0) return launch(kv8_read_kernel<T, HD, false>, ctas, p, st);
    return launch(kv8_read_kernel<T, HD, true>, ctas, p, st);
}

template <typename T>
cudaError_t read_t(const Kv8Read& p, int64_t ctas, cudaStream_t st) {
    if (p.c.head_dim == 64) return read_hd<T, 64>(p, ctas, st);
    if (p.c.head_dim == 96) return read_hd<T, 96>(p, ctas, st);
    return read_hd<T, 128>(p, ctas, st);
}

// Units to launch: n consecutive positions touch at most (n + page - 2) / page + 1 pages wherever they begin, all
// sequences together two each beside those that their rows fill.  A unit without rows costs 2 ns (one with rows
// about 20), counting 3 to 18 % of a launch: units are counted where that launches less than half as many.
int64_t units_of(int n_seq, int n_tokens, int most, int page, int* units) {
    const int64_t each = ((int64_t)std::min(most, n_tokens) + page - 2) / page + 1;
    const int64_t straight = n_seq * each, listed = n_tokens / page + (int64_t)2 * n_seq;
    *units = straight <= 2 * listed ? (int)each : 0;
    return *units ? straight : listed;
}

}  // namespace

cudaError_t launch_kv8_append(int type, Kv8Append p, cudaStream_t st) {
    const int64_t ctas = units_of(p.c.n_seq, p.n_tokens, p.max_new, p.c.page, &p.units) * p.c.n_kv * (p.q_out ? 2 : 1);
    if (type == TPTC_TYPE_F16) return append_t<__half>(p, ctas, st);
    if (type == TPTC_TYPE_BF16) return append_t<__nv_bfloat16>(p, ctas, st);
    return append_t<float>(p, ctas, st);
}

cudaError_t launch_kv8_read(int type, Kv8Read p, cudaStream_t st) {
    // one round of loads per CTA
    p.heads_per_cta = std::max(1, std::min(p.c.n_kv, kReadLoads * kThreads * 16 / (p.c.page * p.c.head_dim)));
    const int64_t ctas =
        units_of(p.c.n_seq, p.n_tokens, p.max_rows, p.c.page, &p.units) * ceil_div(p.c.n_kv, p.heads_per_cta);
    if (type == TPTC_TYPE_F16) return read_t<__half>(p, ctas, st);
    if (type == TPTC_TYPE_BF16) return read_t<__nv_bfloat16>(p, ctas, st);
    return read_t<float>(p, ctas, st);
}

cudaError_t serve_init_device() {
    cudaError_t e = logprobs_init_device();
    if (e == cudaSuccess) e = kv8_attn_init_device();
    if (e == cudaSuccess) e = attn_packed_init_device();
    return e;
}

}  // namespace tptc
