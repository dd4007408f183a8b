// The 8-bit paged K/V cache: rows quantised into pages (wk_kv8_store) and the
// attention of single tokens over it (wk_kv8_attention).
//
// Layout: kpool / vpool [pages][kv_heads][64 tokens][head_dim] e4m3 codes,
// kscale / vscale [pages][kv_heads] fp32; value = code * scale.  The scale of a
// page and head is the smallest power of two s with max |x| <= 448 s over the
// tokens that were written to it.  e4m3 is a floating format: above its
// subnormals a code's relative step does not depend on the scale, so a power of
// two loses nothing against max / 448, and buys two things: x / s is exact (one
// rounding per value, to the code), and when a later token outgrows the scale of
// an open page the codes that it holds move to the new scale exactly unless they
// fall into the subnormals.
#include <cuda_fp8.h>

#include "common.cuh"
#include "wukong_ext.h"
#include "wukong_internal.cuh"

namespace wk {

namespace {

constexpr int kKv8Page = 64;
constexpr int kMinScaleExp = -100;  // scale exponent of a page of zeros

// ------------------------------------------------------------------ store
struct Kv8Store {
    uint8_t *pool[2];        // K, V
    float *scale[2];
    int n_pages;
    const void *x[2];        // K, V rows
    long rs[2];              // their row strides in elements
    const int *starts, *ctx; // [n + 1], [n]
    int n, rows;
    const int *table;
    int max_pages, kv_heads;
};

// The smallest power of two s with amax <= 448 s = 1.75 * 2^8 s, from the bits
// of amax = m 2^e, m in [1, 2): 2^(e - 8), twice that when m > 1.75.
__device__ __forceinline__ float scale_for(float amax) {
    const uint32_t b = __float_as_uint(amax);
    const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u);
    return __uint_as_float((uint32_t)(max(e, kMinScaleExp) + 127) << 23);
}

__device__ __forceinline__ float finite_abs(float v) {
    const float a = fabsf(v);
    return a < INFINITY ? a : 0.f;  // infinities saturate, NaN stays NaN; neither sets the scale
}

// Eight 16-bit values from p; VEC: p is 16-byte aligned.
template <typename T, bool VEC> __device__ __forceinline__ void load8(const T *p, float (&v)[8]) {
    if (VEC) {
        const uint4 u = *reinterpret_cast<const uint4 *>(p);
        const T *t = reinterpret_cast<const T *>(&u);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = to_float(t[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = to_float(p[j]);
    }
}

// One CTA per (page that the call writes, K/V head): threads 0..127 take K,
// 128..255 V.  The page's new rows stay in registers between the maximum and
// the rounding, so each is read once.
template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(256) kv8_store_kernel(Kv8Store a) {
    constexpr int kChunks = D / 8;               // 8-element chunks per row
    constexpr int kRows = 128 / kChunks;         // rows per pass of 128 threads
    constexpr int kPasses = kKv8Page / kRows;
    __shared__ int s_units[8];
    __shared__ int s_found[5];  // sequence, page index, first row, tokens, first offset
    __shared__ float s_max[8];
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    const int unit = blockIdx.x, head = blockIdx.y;
    if (tid == 0) s_found[0] = -1;
    pdl_wait();
    pdl_trigger();
    // the sequence and page of this CTA: a scan over the pages that each sequence's new tokens touch
    int before = 0;
    for (int i0 = 0; i0 < a.n; i0 += 256) {
        const int i = i0 + tid;
        int r0 = 0, add = 0, ctx = 0, u = 0;
        if (i < a.n) {
            r0 = min(max(a.starts[i], 0), a.rows);
            add = min(max(a.starts[i + 1], r0), a.rows) - r0;
            ctx = max(a.ctx[i], 0);
            if (add > 0) u = (ctx % kKv8Page + add + kKv8Page - 1) / kKv8Page;
        }
        int in = u;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, in, o);
            if (lane >= o) in += v;
        }
        __syncthreads();
        if (lane == 31) s_units[wid] = in;
        __syncthreads();
        int first = before + in - u;
#pragma unroll
        for (int w = 0; w < 8; ++w) {
            if (w < wid) first += s_units[w];
            before += s_units[w];
        }
        if (unit >= first && unit < first + u) {
            const int k = unit - first;                           // its k-th touched page
            const int lo = k ? k * kKv8Page - ctx % kKv8Page : 0;  // tokens before this page
            const int off = k ? 0 : ctx % kKv8Page;
            s_found[0] = i;
            s_found[1] = ctx / kKv8Page + k;
            s_found[2] = r0 + lo;
            s_found[3] = min(kKv8Page - off, add - lo);
            s_found[4] = off;
        }
        if (unit < before) break;
    }
    __syncthreads();
    if (s_found[0] < 0 || s_found[1] >= a.max_pages) return;
    const int row0 = s_found[2], m = s_found[3], off = s_found[4];
    const int page = a.table[(long)s_found[0] * a.max_pages + s_found[1]];
    if (page < 0 || page >= a.n_pages) return;
    const int kv = tid >> 7, t = tid & 127;
    const int c = t % kChunks, r = t / kChunks;
    const T *x = reinterpret_cast<const T *>(a.x[kv]) + (long)row0 * a.rs[kv] + head * D + c * 8;
    float v[kPasses][8];
    float amax = 0.f;
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
        const int j = p * kRows + r;
        if (j < m) {
            load8<T, VEC>(x + (long)j * a.rs[kv], v[p]);
#pragma unroll
            for (int e = 0; e < 8; ++e) amax = fmaxf(amax, finite_abs(v[p][e]));
        }
    }
    const long ps = (long)page * a.kv_heads + head;
    const float old = off ? a.scale[kv][ps] : 0.f;
    amax = warp_max(amax);
    if (lane == 0) s_max[wid] = amax;
    __syncthreads();
    amax = fmaxf(fmaxf(s_max[4 * kv], s_max[4 * kv + 1]), fmaxf(s_max[4 * kv + 2], s_max[4 * kv + 3]));
    const float scale = fmaxf(old, scale_for(amax));
    const float inv = 1.0f / scale;  // a power of two: exact
    uint8_t *dst = a.pool[kv] + (size_t)ps * (kKv8Page * D);
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
        const int j = p * kRows + r;
        if (j < m) {
            uint2 o;
            __nv_fp8x2_storage_t *w = reinterpret_cast<__nv_fp8x2_storage_t *>(&o);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                w[e] = __nv_cvt_float2_to_fp8x2(make_float2(v[p][2 * e] * inv, v[p][2 * e + 1] * inv), __NV_SATFINITE,
                                                __NV_E4M3);
            *reinterpret_cast<uint2 *>(dst + (off + j) * D + c * 8) = o;
        }
    }
    if (off && scale != old) {  // the tokens that the page held move to the new scale
        const float ratio = old * inv;
        for (int i = t; i < off * D / 2; i += 128) {
            __nv_fp8x2_storage_t *w = reinterpret_cast<__nv_fp8x2_storage_t *>(dst) + i;
            const __half2 h(__nv_cvt_fp8x2_to_halfraw2(*w, __NV_E4M3));
            const float2 f = __half22float2(h);
            *w = __nv_cvt_float2_to_fp8x2(make_float2(f.x * ratio, f.y * ratio), __NV_SATFINITE, __NV_E4M3);
        }
    }
    if (t == 0) a.scale[kv][ps] = scale;
}

// ------------------------------------------------------------------ attention
struct Kv8Attn {
    void *out;
    long out_rs;
    const void *q;
    long q_rs;
    const uint8_t *kpool, *vpool;
    const float *kscale, *vscale;
    int n_pages;
    const int *table;
    int n_seqs, max_pages;
    const int *seq, *pos;
    int heads, kv_heads;
    float scale;
};

__device__ __forceinline__ float e4m3_to_float(uint8_t b) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(b, __NV_E4M3)));
}

// One CTA per (row, query head), 128 threads: a thread scores one key of each
// block of 128, then owns one dimension of the output.
template <typename T, int D>
__global__ void __launch_bounds__(128) kv8_attn_kernel(Kv8Attn a) {
    __shared__ float s_q[D], s_p[128], s_w[4];
    __shared__ int s_page[2];
    const int row = blockIdx.y, h = blockIdx.x, tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    const int kh = h / (a.heads / a.kv_heads);
    pdl_wait();
    pdl_trigger();
    const int seq = a.seq[row];
    const long len = seq >= 0 && seq < a.n_seqs
                         ? min((long)a.pos[row] + 1, (long)a.max_pages * kKv8Page) : 0;
    if (tid < D) s_q[tid] = to_float(reinterpret_cast<const T *>(a.q)[row * a.q_rs + h * D + tid]) * a.scale;
    float m = -INFINITY, l = 0.f, o = 0.f;
    for (long k0 = 0; k0 < len; k0 += 128) {
        __syncthreads();
        if (tid < 2) {
            const long p = k0 / kKv8Page + tid;
            const int page = p < a.max_pages ? a.table[(long)seq * a.max_pages + p] : -1;
            s_page[tid] = page < a.n_pages ? page : -1;
        }
        __syncthreads();
        float s = -INFINITY;
        const int page = s_page[tid / kKv8Page];
        if (k0 + tid < len && page >= 0) {
            const long ps = (long)page * a.kv_heads + kh;
            const uint8_t *k = a.kpool + (ps * kKv8Page + tid % kKv8Page) * D;
            float dot = 0.f;
            for (int d = 0; d < D; ++d) dot += s_q[d] * e4m3_to_float(k[d]);
            s = dot * a.kscale[ps];
        }
        float bm = warp_max(s);
        if (lane == 0) s_w[wid] = bm;
        __syncthreads();
        const float mn = fmaxf(m, fmaxf(fmaxf(s_w[0], s_w[1]), fmaxf(s_w[2], s_w[3])));
        const float p = s == -INFINITY ? 0.f : expf(s - mn);
        s_p[tid] = p;
        __syncthreads();
        const float ps_ = warp_sum(p);
        if (lane == 0) s_w[wid] = ps_;
        __syncthreads();
        const float c = mn == -INFINITY ? 1.f : expf(m - mn);
        l = l * c + (s_w[0] + s_w[1] + s_w[2] + s_w[3]);
        o *= c;
        m = mn;
        if (tid < D) {
            for (int b = 0; b < 2; ++b) {
                if (s_page[b] < 0) continue;
                const long ps = (long)s_page[b] * a.kv_heads + kh;
                const uint8_t *v = a.vpool + ps * kKv8Page * D + tid;
                const int n = (int)min(len - k0 - b * kKv8Page, (long)kKv8Page);
                float acc = 0.f;
                for (int j = 0; j < n; ++j) acc += s_p[b * kKv8Page + j] * e4m3_to_float(v[j * D]);
                o += acc * a.vscale[ps];
            }
        }
    }
    if (tid < D)
        reinterpret_cast<T *>(a.out)[row * a.out_rs + h * D + tid] = from_float<T>(l > 0.f || l != l ? o / l : 0.f);
}

template <typename T, int D> cudaError_t launch_store(const Kv8Store &a, int units, cudaStream_t s) {
    const bool vec = ((uintptr_t)a.x[0] % 16) == 0 && ((uintptr_t)a.x[1] % 16) == 0 && a.rs[0] % 8 == 0 &&
                     a.rs[1] % 8 == 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(units, a.kv_heads);
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = g_rt.pdl ? 1 : 0;
    return vec ? cudaLaunchKernelEx(&cfg, kv8_store_kernel<T, D, true>, a)
               : cudaLaunchKernelEx(&cfg, kv8_store_kernel<T, D, false>, a);
}

template <typename T, int D> cudaError_t launch_attn(const Kv8Attn &a, int rows, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.heads, rows);
    cfg.blockDim = dim3(128);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = g_rt.pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kv8_attn_kernel<T, D>, a);
}

}  // namespace

}  // namespace wk

using namespace wk;

extern "C" {

int wk_kv8_store(void *kpool, void *vpool, float *kscale, float *vscale, int n_pages, const void *k, long k_rs,
                 const void *v, long v_rs, const int *starts, const int *ctx, int n, int rows, const int *block_table,
                 int max_pages, int kv_heads, int head_dim, int dtype) {
    if (n < 0 || rows < 0 || n_pages < 1 || max_pages < 1 || kv_heads < 1 || kv_heads > 65535)
        return fail("wk_kv8_store: bad sizes");
    if (head_dim != 64 && head_dim != 128) return fail("wk_kv8_store: head_dim %d (64 or 128)", head_dim);
    if (dtype != kF16 && dtype != kBF16) return fail("wk_kv8_store: dtype %d (F16 or BF16)", dtype);
    if (n == 0 || rows == 0) return 0;
    if (!kpool || !vpool || !kscale || !vscale || !k || !v || !starts || !ctx || !block_table)
        return fail("wk_kv8_store: null argument");
    if (k_rs < (long)kv_heads * head_dim || v_rs < (long)kv_heads * head_dim)
        return fail("wk_kv8_store: row stride below kv_heads * head_dim");
    if (((uintptr_t)kpool % 16) || ((uintptr_t)vpool % 16)) return fail("wk_kv8_store: pools must be 16-byte aligned");
    if (g_rt.device < 0) return fail("wk_kv8_store: cuda_init() has not been called");
    DeviceGuard guard;
    Kv8Store a{{(uint8_t *)kpool, (uint8_t *)vpool}, {kscale, vscale}, n_pages, {k, v}, {k_rs, v_rs}, starts, ctx, n,
               rows, block_table, max_pages, kv_heads};
    // pages touched: at most one per row, and at most ceil((63 + add) / 64) per sequence
    const long long most = (long long)rows / kKv8Page + 2ll * n;
    const int units = (int)(most < rows ? most : rows);
    cudaStream_t s = stream();
    cudaError_t e;
    if (dtype == kF16)
        e = head_dim == 64 ? launch_store<__half, 64>(a, units, s) : launch_store<__half, 128>(a, units, s);
    else
        e = head_dim == 64 ? launch_store<__nv_bfloat16, 64>(a, units, s) : launch_store<__nv_bfloat16, 128>(a, units, s);
    if (e != cudaSuccess) return fail("wk_kv8_store: %s", cudaGetErrorString(e));
    return 0;
}

long long wk_kv8_attention_ws(int rows, int max_len, int n_heads, int kv_heads, int head_dim) {
    (void)rows, (void)max_len, (void)n_heads, (void)kv_heads, (void)head_dim;
    return 0;
}

int wk_kv8_attention(void *out, long out_rs, const void *q, long q_rs, const void *kpool, const void *vpool,
                     const float *kscale, const float *vscale, int n_pages, const int *block_table, int n_seqs,
                     int max_pages, const int *seq, const int *pos, int rows, int max_len, int n_heads, int kv_heads,
                     int head_dim, int dtype, void *ws, long long ws_bytes) {
    if (rows < 0 || rows > 65535 || n_pages < 1 || n_seqs < 1 || max_pages < 1 || max_len < 0 || ws_bytes < 0)
        return fail("wk_kv8_attention: bad sizes");
    if (kv_heads < 1 || n_heads < 1 || n_heads % kv_heads) return fail("wk_kv8_attention: %d heads over %d", n_heads, kv_heads);
    if (head_dim != 64 && head_dim != 128) return fail("wk_kv8_attention: head_dim %d (64 or 128)", head_dim);
    if (dtype != kF16 && dtype != kBF16) return fail("wk_kv8_attention: dtype %d (F16 or BF16)", dtype);
    if (rows == 0) return 0;
    if (!out || !q || !kpool || !vpool || !kscale || !vscale || !block_table || !seq || !pos)
        return fail("wk_kv8_attention: null argument");
    if (q_rs < (long)n_heads * head_dim || out_rs < (long)n_heads * head_dim)
        return fail("wk_kv8_attention: row stride below n_heads * head_dim");
    if (((uintptr_t)kpool % 16) || ((uintptr_t)vpool % 16))
        return fail("wk_kv8_attention: pools must be 16-byte aligned");
    if (g_rt.device < 0) return fail("wk_kv8_attention: cuda_init() has not been called");
    DeviceGuard guard;
    Kv8Attn a{out, out_rs, q, q_rs, (const uint8_t *)kpool, (const uint8_t *)vpool, kscale, vscale, n_pages,
              block_table, n_seqs, max_pages, seq, pos, n_heads, kv_heads, 1.0f / sqrtf((float)head_dim)};
    cudaStream_t s = stream();
    cudaError_t e;
    if (dtype == kF16)
        e = head_dim == 64 ? launch_attn<__half, 64>(a, rows, s) : launch_attn<__half, 128>(a, rows, s);
    else
        e = head_dim == 64 ? launch_attn<__nv_bfloat16, 64>(a, rows, s) : launch_attn<__nv_bfloat16, 128>(a, rows, s);
    if (e != cudaSuccess) return fail("wk_kv8_attention: %s", cudaGetErrorString(e));
    (void)ws;
    return 0;
}

}  // extern "C"
