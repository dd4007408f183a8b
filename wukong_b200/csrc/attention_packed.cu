// Causal attention with grouped heads over packed sequences (wk_attention_packed).
//
// Sequence i has query rows [q_starts[i], q_starts[i+1]) and key rows
// [k_starts[i], k_starts[i+1]); its queries are the last of its keys, so query
// row j of Lq sees the keys 0 .. Lk - Lq + j:
//   o = sum_k softmax_k(q . k / sqrt(d)) v
#include "common.cuh"
#include "wukong_ext.h"
#include "wukong_internal.cuh"

namespace wk {

namespace {

struct PackedArgs {
    void *out;
    long out_rs;
    const void *q, *k, *v;
    long q_rs, k_rs, v_rs;
    const int *q_starts, *k_starts;
    int n, q_rows, k_rows, heads, kv_heads;
    float scale;
};

// One CTA per (query row, head), 128 threads: a thread scores one key of each
// block of 128, then owns one dimension of the output.
template <typename T, int D>
__global__ void __launch_bounds__(128) attn_packed_rows_kernel(PackedArgs a) {
    __shared__ float s_q[D], s_p[128], s_w[4];
    __shared__ int s_seq[1];
    const int h = blockIdx.y, tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    const int row = blockIdx.x;
    const int kh = h / (a.heads / a.kv_heads);
    pdl_wait();
    pdl_trigger();
    // the sequence that holds this row (starts ascend; an empty sequence holds none)
    if (tid == 0) s_seq[0] = -1;
    __syncthreads();
    for (int i = tid; i < a.n; i += 128)
        if (row >= a.q_starts[i] && row < a.q_starts[i + 1]) s_seq[0] = i;
    __syncthreads();
    const int seq = s_seq[0];
    if (seq < 0) return;
    const int q0 = a.q_starts[seq], ql = a.q_starts[seq + 1] - q0;
    const int k0 = min(max(a.k_starts[seq], 0), a.k_rows);
    const int kl = min(max(a.k_starts[seq + 1], k0), a.k_rows) - k0;
    const int len = min(kl, kl - ql + (row - q0) + 1);
    if (tid < D) s_q[tid] = to_float(reinterpret_cast<const T *>(a.q)[row * a.q_rs + h * D + tid]) * a.scale;
    float m = -INFINITY, l = 0.f, o = 0.f;
    for (int j0 = 0; j0 < len; j0 += 128) {
        __syncthreads();
        float s = -INFINITY;
        if (j0 + tid < len) {
            const T *k = reinterpret_cast<const T *>(a.k) + (long)(k0 + j0 + tid) * a.k_rs + kh * D;
            float dot = 0.f;
            for (int d = 0; d < D; ++d) dot += s_q[d] * to_float(k[d]);
            s = dot;
        }
        const float bm = warp_max(s);
        if (lane == 0) s_w[wid] = bm;
        __syncthreads();
        const float mn = fmaxf(m, fmaxf(fmaxf(s_w[0], s_w[1]), fmaxf(s_w[2], s_w[3])));
        const float p = s == -INFINITY ? 0.f : expf(s - mn);
        s_p[tid] = p;
        __syncthreads();
        const float sum = warp_sum(p);
        if (lane == 0) s_w[wid] = sum;
        __syncthreads();
        const float c = mn == -INFINITY ? 1.f : expf(m - mn);
        l = l * c + (s_w[0] + s_w[1] + s_w[2] + s_w[3]);
        o *= c;
        m = mn;
        if (tid < D) {
            const T *v = reinterpret_cast<const T *>(a.v) + (long)(k0 + j0) * a.v_rs + kh * D + tid;
            const int n = min(len - j0, 128);
            for (int j = 0; j < n; ++j) o += s_p[j] * to_float(v[(long)j * a.v_rs]);
        }
    }
    if (tid < D)
        reinterpret_cast<T *>(a.out)[row * a.out_rs + h * D + tid] = from_float<T>(l > 0.f || l != l ? o / l : 0.f);
}

template <typename T, int D> cudaError_t launch_rows(const PackedArgs &a, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.q_rows, a.heads);
    cfg.blockDim = dim3(128);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = g_rt.pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, attn_packed_rows_kernel<T, D>, a);
}

}  // namespace

}  // namespace wk

using namespace wk;

extern "C" {

int wk_attention_packed(void *out, long out_rs, const void *q, long q_rs, const void *k, long k_rs, const void *v,
                        long v_rs, const int *q_starts, const int *k_starts, int n, int q_rows, int k_rows,
                        int n_heads, int kv_heads, int head_dim, int dtype) {
    if (n < 0 || q_rows < 0 || k_rows < 0) return fail("wk_attention_packed: bad sizes");
    if (kv_heads < 1 || n_heads < 1 || n_heads % kv_heads || n_heads > 65535)
        return fail("wk_attention_packed: %d heads over %d", n_heads, kv_heads);
    if (head_dim != 64 && head_dim != 128) return fail("wk_attention_packed: head_dim %d (64 or 128)", head_dim);
    if (dtype != kF16 && dtype != kBF16) return fail("wk_attention_packed: dtype %d (F16 or BF16)", dtype);
    if (n == 0 || q_rows == 0) return 0;
    if (!out || !q || !q_starts || !k_starts || (k_rows && (!k || !v)))
        return fail("wk_attention_packed: null argument");
    const long qw = (long)n_heads * head_dim, kw = (long)kv_heads * head_dim;
    if (out_rs < qw || q_rs < qw || k_rs < kw || v_rs < kw)
        return fail("wk_attention_packed: row stride below heads * head_dim");
    if (g_rt.device < 0) return fail("wk_attention_packed: cuda_init() has not been called");
    DeviceGuard guard;
    PackedArgs a{out, out_rs, q, k, v, q_rs, k_rs, v_rs, q_starts, k_starts, n, q_rows, k_rows, n_heads, kv_heads,
                 1.0f / sqrtf((float)head_dim)};
    cudaStream_t s = stream();
    cudaError_t e;
    if (dtype == kF16)
        e = head_dim == 64 ? launch_rows<__half, 64>(a, s) : launch_rows<__half, 128>(a, s);
    else
        e = head_dim == 64 ? launch_rows<__nv_bfloat16, 64>(a, s) : launch_rows<__nv_bfloat16, 128>(a, s);
    if (e != cudaSuccess) return fail("wk_attention_packed: %s", cudaGetErrorString(e));
    return 0;
}

}  // extern "C"
