// Causal attention with grouped heads over packed sequences (wk_attention_packed).
//
// Sequence i has query rows [q_starts[i], q_starts[i+1]) and key rows
// [k_starts[i], k_starts[i+1]); its queries are the last of its keys, so query
// row j of Lq sees the keys 0 .. Lk - Lq + j:
//   o = sum_k softmax_k(q . k / sqrt(d)) v
#include <cudaTypedefs.h>

#include <type_traits>

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
    bool out4;  // out's rows are 4-byte aligned
    int reach;  // sequences of up to so many keys are the short kernel's, longer ones the tcgen05 kernel's
    int longer; // how many longer ones there can be
};

// Softmax weights are multiplied with V in V's type.  fp16 is exact to 2^-25 at the least, so
// its weights go in as 2^bias p, at the top of its range: O and the sum l share the factor.
// `lead`: log2 of how far the reference of p may fall behind the largest score (p <= 2^lead).
// With bias 0 the keys behind one that leads them by 18 and has V = 0 counted for nothing; with
// 9 a p down to 2^-23 is rounded relative to itself, a smaller one to 2^-34.  (24 prompts of
// 1 to 1500 tokens, 16 / 4 heads of 64: 39.6 us, as with a lead of 8; 1 % more with 5, 8 % with 4.)
// References are rounded up, so that 2^(lead + bias) bounds the weights for scores up to 10^8.
template <typename T> struct PkWeight {
    static constexpr float lead = 6.f, bias = 9.f;
};
// bf16 has fp32's range: 2^bias keeps the sums over up to 2^24 keys below V's own largest value.
template <> struct PkWeight<__nv_bfloat16> {
    static constexpr float lead = 8.f, bias = -32.f;
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
    // the sequence that holds this row (starts ascend; an empty sequence holds none); starts beyond the
    // rows count as the end of them, as in the other kernels
    if (tid == 0) s_seq[0] = -1;
    __syncthreads();
    for (int i = tid; i < a.n; i += 128)
        if (row >= a.q_starts[i] && row < a.q_starts[i + 1]) s_seq[0] = i;
    __syncthreads();
    const int seq = s_seq[0];
    if (seq < 0) return;
    const int q0 = max(a.q_starts[seq], 0), ql = min(a.q_starts[seq + 1], a.q_rows) - q0;
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
        const float p = s == -INFINITY ? 0.f : expf(s - mn) * 0x1p-24f;  // (sums stay below V's largest value)
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

// ------------------------------------------------------------------ short sequences
// A CTA takes 64 rows of one sequence and K/V head, a row being a position and one
// of the G heads of the group (heads inner, so no row is empty but at a sequence's end);
// a warp takes 16 of them, with S, P and O in mma.sync fragments:
//   S = Q K^T     P = exp2(c (S - m) + b)     O += P V     l += row sums of P before rounding
// Blocks of 64 keys come through two stages of cp.async.  The contraction of Q K^T runs
// over dims in the order in which 16-byte pieces of a row fall to the four lanes
// of a row group, so Q goes from global memory straight into its fragments and a K
// fragment is one 16-byte read.  m is the running maximum itself, so b = lead + bias: 15 in
// fp16, -24 in bf16.
// Latency bounds it: unit -> Q, K, V -> S -> softmax -> O.  Small CTAs, several to an SM, and
// no tensor memory, barriers or maps to set up are what it has over the tcgen05 kernel: 100
// sequences of 40 tokens, 16 / 4 heads of 64, take 10.5 us instead of 22.0.  A further block
// of 64 keys costs 1.6 us with D = 128, so sequences of more than `reach` keys are not for it
// (where they begin to cost more stands at the launch).
// A row whose result is not finite is computed again over the keys that it sees alone,
// for a masked key has p = 0, and 0 * NaN is NaN.
__device__ __forceinline__ float pk_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <int D> struct ShLayout {
    static constexpr int kKeys = 64;
    static constexpr int kPitchK = 2 * D + 64, kPitchV = 2 * D + 16;  // bytes; reads free of bank conflicts
    static constexpr int kK = kKeys * kPitchK, kStage = kK + kKeys * kPitchV;
    static constexpr int kSmem = 2 * kStage;
};

template <typename T> __device__ __forceinline__ uint32_t sh_pack(float lo, float hi);
template <> __device__ __forceinline__ uint32_t sh_pack<__half>(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <> __device__ __forceinline__ uint32_t sh_pack<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <typename T>
__device__ __forceinline__ void sh_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    if (std::is_same<T, __half>::value)
        mma_f16(c, a0, a1, a2, a3, b0, b1);
    else
        mma_bf16(c, a0, a1, a2, a3, b0, b1);
}
__device__ __forceinline__ void sh_cp16(uint32_t dst, const void *src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

template <typename T, int D>
__global__ void __launch_bounds__(128, D == 128 ? 3 : 4) attn_packed_short_kernel(PackedArgs a) {
    using L = ShLayout<D>;
    constexpr int NC = D / 32;  // 16-byte pieces of a row per lane
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ int s_unit[6];  // found, q0, ql, k0, kl, first row
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int kvh = blockIdx.x, G = a.heads / a.kv_heads;
    const int unit = gridDim.y - 1 - blockIdx.y;  // a long prompt's last rows, which see most, start first
    if (tid == 0) s_unit[0] = 0;
    __syncthreads();
    pdl_wait();
    pdl_trigger();
    // Sequence i has room for its units from base(i) = min(q_starts, G q_starts / 64 + i) to
    // base(i + 1) (G <= 64), so it is found by comparisons alone.
    auto start = [&](int i) -> int { return min(max(a.q_starts[i], 0), a.q_rows); };
    auto base = [&](int r, int i) -> int { return (int)min((long)r, (long)r * G / 64 + i); };
    int lo = 0, n = a.n;
    while (n > 128) {
        const int st = (n + 127) / 128, i = lo + tid * st;
        const int c = __syncthreads_count(tid * st < n && base(start(i), i) <= unit);
        if (c == 0) return;
        lo += (c - 1) * st;
        n = min(st, n - (c - 1) * st);
    }
    if (tid < n) {
        const int i = lo + tid, r0 = start(i), r1 = max(start(i + 1), r0), k0 = a.k_starts[i], k1 = a.k_starts[i + 1];
        const int k = unit - base(r0, i);
        if (k >= 0 && unit < base(r1, i + 1) && (long)k * 64 < (long)(r1 - r0) * G) {
            s_unit[1] = r0;
            s_unit[2] = r1 - r0;
            s_unit[3] = min(max(k0, 0), a.k_rows);
            s_unit[4] = min(max(k1, s_unit[3]), a.k_rows) - s_unit[3];
            s_unit[5] = k * 64;
            s_unit[0] = s_unit[4] <= a.reach;
        }
    }
    __syncthreads();
    if (!s_unit[0]) return;
    const int q0 = s_unit[1], ql = s_unit[2], k0 = s_unit[3], kl = s_unit[4], x0 = s_unit[5];
    const int rows = (int)min((long)ql * G - x0, 64l);  // of this unit
    const int p0 = x0 / G, h0 = x0 - p0 * G;            // position and head of its first row
    auto seen = [&](int r) -> int { return max(0, min(kl, kl - ql + p0 + (h0 + r) / G + 1)); };  // keys of row r
    const int blocks = (seen(rows - 1) + L::kKeys - 1) / L::kKeys;

    const uint32_t smem = smem_u32(sm);
    const T *kp = reinterpret_cast<const T *>(a.k) + (long)k0 * a.k_rs + kvh * D;
    const T *vp = reinterpret_cast<const T *>(a.v) + (long)k0 * a.v_rs + kvh * D;
    auto load = [&](int b) {
        constexpr int per = D / 8;  // 16-byte pieces of a row
        const uint32_t st = smem + (b & 1) * L::kStage;
#pragma unroll
        for (int x = 0; x < L::kKeys * per / 128; ++x) {
            const int j = (tid + x * 128) / per, c = (tid + x * 128) % per, key = b * L::kKeys + j;
            const int row = min(key, kl - 1), bytes = key < kl ? 16 : 0;  // rows behind the sequence: zeros
            sh_cp16(st + j * L::kPitchK + c * 16, kp + row * a.k_rs + c * 8, bytes);
            sh_cp16(st + L::kK + j * L::kPitchV + c * 16, vp + row * a.v_rs + c * 8, bytes);
        }
    };
    if (blocks > 0) load(0);
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (blocks > 1) load(1);
    asm volatile("cp.async.commit_group;" ::: "memory");

    // this thread's rows: r, r + 8
    const int r = warp * 16 + g;
    uint4 q[2][NC];
    int len[2];
    long at[2];  // of the row, in heads of the unit's K/V head
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int x = r + 8 * i, p = (h0 + x) / G, h = h0 + x - p * G;
        len[i] = x < rows ? seen(x) : 0;
        const T *src = reinterpret_cast<const T *>(a.q) + (long)(q0 + p0 + p) * a.q_rs + (long)(kvh * G + h) * D + t * 8;
        at[i] = (long)(q0 + p0 + p) * a.out_rs + (long)(kvh * G + h) * D;
#pragma unroll
        for (int c = 0; c < NC; ++c)
            q[i][c] = x < rows ? *reinterpret_cast<const uint4 *>(src + c * 32) : make_uint4(0, 0, 0, 0);
    }
    const int wrows = min(rows - warp * 16, 16);  // of this warp
    const int wlast = wrows > 0 ? seen(warp * 16 + wrows - 1) : 0, wfirst = wrows > 0 ? seen(warp * 16) : 0;
    const float c2 = a.scale * 1.4426950408889634f;
    float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = 0.f;

    for (int b = 0; b < blocks; ++b) {
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncthreads();
        const int left = wlast - b * L::kKeys;  // keys from here on that a row of the warp sees
        if (left > 0) {
            const uint8_t *ks = sm + (b & 1) * L::kStage;
            const uint32_t vs = smem + (b & 1) * L::kStage + L::kK;
            float s[8][4];
#pragma unroll
            for (int hb = 0; hb < 8; hb += 4) {  // 32 keys: four sums under way at a time
#pragma unroll
                for (int nt = hb; nt < hb + 4; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[nt][e] = 0.f;
                if (hb * 8 < left) {
#pragma unroll
                    for (int c = 0; c < NC; ++c) {
                        uint4 k[4];
#pragma unroll
                        for (int nt = 0; nt < 4; ++nt)
                            k[nt] = *reinterpret_cast<const uint4 *>(ks + ((hb + nt) * 8 + g) * L::kPitchK + (t + 4 * c) * 16);
#pragma unroll
                        for (int nt = 0; nt < 4; ++nt)
                            sh_mma<T>(s[hb + nt], q[0][c].x, q[1][c].x, q[0][c].y, q[1][c].y, k[nt].x, k[nt].y);
#pragma unroll
                        for (int nt = 0; nt < 4; ++nt)
                            sh_mma<T>(s[hb + nt], q[0][c].z, q[1][c].z, q[0][c].w, q[1][c].w, k[nt].z, k[nt].w);
                    }
                }
            }
            if (b * L::kKeys + L::kKeys > wfirst) {
#pragma unroll
                for (int nt = 0; nt < 8; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (b * L::kKeys + nt * 8 + 2 * t + (e & 1) >= len[e >> 1]) s[nt][e] = -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float mx = m[i];
#pragma unroll
                for (int nt = 0; nt < 8; ++nt) mx = fmaxf(mx, fmaxf(s[nt][2 * i], s[nt][2 * i + 1]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float f = mx == m[i] ? 1.f : pk_ex2((m[i] - mx) * c2);
                const float ref = mx == -INFINITY ? 0.f : __fmaf_ru(mx, c2, -PkWeight<T>::lead - PkWeight<T>::bias);
                m[i] = mx;
                l[i] *= f;
#pragma unroll
                for (int nt = 0; nt < D / 8; ++nt) o[nt][2 * i] *= f, o[nt][2 * i + 1] *= f;
#pragma unroll
                for (int nt = 0; nt < 8; ++nt) {
                    s[nt][2 * i] = pk_ex2(s[nt][2 * i] * c2 - ref);
                    s[nt][2 * i + 1] = pk_ex2(s[nt][2 * i + 1] * c2 - ref);
                    l[i] += s[nt][2 * i] + s[nt][2 * i + 1];
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j * 16 < left) {
                    const uint32_t a0 = sh_pack<T>(s[2 * j][0], s[2 * j][1]), a1 = sh_pack<T>(s[2 * j][2], s[2 * j][3]);
                    const uint32_t a2 = sh_pack<T>(s[2 * j + 1][0], s[2 * j + 1][1]),
                                   a3 = sh_pack<T>(s[2 * j + 1][2], s[2 * j + 1][3]);
                    const uint32_t vr = vs + (j * 16 + (lane & 15)) * L::kPitchV + (lane >> 4) * 16;
#pragma unroll
                    for (int n4 = 0; n4 < D / 16; n4 += 4) {
                        uint32_t w[4][4];
#pragma unroll
                        for (int nt = 0; nt < 4; ++nt) ldsm_x4_t(vr + (n4 + nt) * 32, w[nt][0], w[nt][1], w[nt][2], w[nt][3]);
#pragma unroll
                        for (int nt = 0; nt < 4; ++nt) {
                            sh_mma<T>(o[2 * (n4 + nt)], a0, a1, a2, a3, w[nt][0], w[nt][1]);
                            sh_mma<T>(o[2 * (n4 + nt) + 1], a0, a1, a2, a3, w[nt][2], w[nt][3]);
                        }
                    }
                }
            }
        }
        __syncthreads();
        if (b + 2 < blocks) load(b + 2);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    uint32_t bad = 0;  // the warp's rows whose result is not finite
    T *out = reinterpret_cast<T *>(a.out);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        const float inv = l[i] > 0.f || l[i] != l[i] ? 1.f / l[i] : 0.f;
        bool fine = true;
#pragma unroll
        for (int nt = 0; nt < D / 8; ++nt) {
            o[nt][2 * i] *= inv;
            o[nt][2 * i + 1] *= inv;
            fine = fine && fabsf(o[nt][2 * i]) < INFINITY && fabsf(o[nt][2 * i + 1]) < INFINITY;
        }
        const uint32_t no = __ballot_sync(0xffffffffu, !fine);
#pragma unroll
        for (int x = 0; x < 8; ++x)
            if (no >> (4 * x) & 15u) bad |= 1u << (x + 8 * i);
        if (r + 8 * i < rows && !(bad >> (g + 8 * i) & 1u)) {
            T *dst = out + at[i] + 2 * t;
#pragma unroll
            for (int nt = 0; nt < D / 8; ++nt) {
                if (a.out4) {
                    *reinterpret_cast<uint32_t *>(dst + nt * 8) = sh_pack<T>(o[nt][2 * i], o[nt][2 * i + 1]);
                } else {
                    dst[nt * 8] = from_float<T>(o[nt][2 * i]);
                    dst[nt * 8 + 1] = from_float<T>(o[nt][2 * i + 1]);
                }
            }
        }
    }
    for (; bad; bad &= bad - 1) {
        const int x = warp * 16 + __ffs(bad) - 1;
        if (x >= rows) break;
        const int p = (h0 + x) / G, h = h0 + x - p * G, len = seen(x);
        const long head = (long)(kvh * G + h) * D;
        const T *qr = reinterpret_cast<const T *>(a.q) + (long)(q0 + p0 + p) * a.q_rs + head;
        float mr = -INFINITY, lr = 0.f, v[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) v[c] = 0.f;
        for (int j = 0; j < len; ++j) {
            float dot = 0.f;
#pragma unroll
            for (int c = 0; c < NC; ++c) dot += to_float(qr[lane + 32 * c]) * to_float(kp[j * a.k_rs + lane + 32 * c]);
            dot = warp_sum(dot) * c2;
            const float mn = fmaxf(mr, dot), f = mr == mn ? 1.f : pk_ex2(mr - mn);
            const float w = dot == -INFINITY ? 0.f : pk_ex2(dot - mn + (PkWeight<T>::lead + PkWeight<T>::bias));
            mr = mn;
            lr = lr * f + w;
#pragma unroll
            for (int c = 0; c < NC; ++c) v[c] = v[c] * f + w * to_float(vp[j * a.v_rs + lane + 32 * c]);
        }
        T *dst = out + (long)(q0 + p0 + p) * a.out_rs + head;
#pragma unroll
        for (int c = 0; c < NC; ++c)
            dst[lane + 32 * c] = from_float<T>(lr > 0.f || lr != lr ? v[c] / lr : 0.f);
    }
}

// ------------------------------------------------------------------ tcgen05 kernel
// A CTA takes one unit: 2 tiles of 128 query rows of one K/V head, a tile being
// PT = 128 / G positions times the G heads of the group (heads inner), so that a
// K/V tile loaded once serves all of them.  Per block of 128 keys and tile t:
//   S_t = Q_t K^T  (TMEM, fp32)       P_t = exp2(c (S_t - m) + b)  (16 bits, over S_t in TMEM)
//   O_t += P_t V   (TMEM, fp32)       l_t += row sums of P_t before rounding
// P is rounded to V's type, which is what the tensor cores multiply V with: at most
// half a step of that type relative to each p, and l_t does not inherit it.
// m is a maximum that is moved, and O_t and l_t scaled, only when it falls more
// than 2^6 (bf16: 2^8) behind the running maximum, so that nearly every block
// skips the pass over O_t.  The first half of a block's
// exponentials is computed against the old maximum before the block's own is
// known, and thrown away in the rare case that it moves.
//   warps 0-3, 4-7   softmax of tile 0, tile 1 (one thread per row), epilogue
//   warp 8           issues the tcgen05.mma
//   warp 9           TMA: Q, then K and V blocks through a ring
//   warps 10, 11     clear what masked keys of V hold (see below)
// While one tile's softmax runs on the CUDA cores, the tensor cores run the
// other tile's P V and its next Q K^T.
//
// A masked key has p = 0, but 0 * NaN is NaN in a product of tiles.  So in the
// blocks that some row of the unit sees in part, warps 10 and 11 set the rows of
// V behind the sequence's end to zero, and every infinity or NaN inside it too,
// noting its key and dimension; rows that do see that key get NaN there.
//
// Where the units are fewer than half the SMs and their keys many, a cluster of CTAs takes
// each, with consecutive shares of its key blocks, and joins O, m and l through distributed
// shared memory.
//
// What bounds it: one block of two tiles takes 3200 to 3400 cycles with D = 128, of
// which the tensor cores run 2048 and the exponentials fill their pipe for 2048;
// the two overlap except where S, P and the barriers between them change hands
// (a barrier's answer waits 150 to 350 cycles behind queued exponentials).  8192 x 32
// heads of 128 over 8: 454 us or 1210 TFLOP/s by itself, 510 to 520 us in calls over
// seconds, under the power cap; behind a long context the tensor pipe is active 61 % of
// the time.  Measured and not kept: exponentials on the FMA pipe by a polynomial for 1/8
// to 1/2 of the keys (no faster), an issuing warp per tile (the tiles fall in phase, 16 %
// slower), P in TMEM columns of its own for D = 64 (the same time), one tile per CTA and
// two CTAs per SM (25 % slower at 8192), persistent CTAs over units (24 ragged prompts
// 5 % faster, one of 8192 3 % slower).
constexpr int kPkThreads = 384;
constexpr int kPkRegs = 168;  // registers per thread at launch
constexpr int kPkKeys = 128;  // keys per block
constexpr int kPkGridY = 32768;  // units go over the grid's y, then z

template <int D> struct PkLayout {
    static constexpr int kTile = 128 * D * 2;                 // bytes of a Q tile or a K / V block
    static constexpr int kStages = D == 128 ? 5 : 8;
    static constexpr size_t kQ = 0;
    static constexpr size_t kRing = 2 * (size_t)kTile;
    static constexpr size_t kBars = kRing + (size_t)kStages * kTile;
};

struct PkUnit {
    int valid;
    int q0, ql, k0, kl;  // the sequence's first rows and their counts
    int j0;              // first query of the unit
};

template <int D> struct PkBars {
    uint64_t q_full, kv_full[PkLayout<D>::kStages], kv_empty[PkLayout<D>::kStages];
    uint64_t s_full[2], p_half[2], p_full[2], o_full[2];
    uint64_t v_raw[4], v_clean[4];  // V blocks that are seen in part: loaded, cleared (the ring holds at most 4)
    uint32_t tmem;
    PkUnit unit;
    int units[kPkThreads / 32];
    int bad;           // a non-finite V in a masked block
    __align__(16) int bad_key[D];  // first key that holds one, per dimension
};

struct PkMaps {
    CUtensorMap q, k, v;
};

__device__ __forceinline__ void pk_tma3(void *dst, const CUtensorMap *map, int x, int y, int z, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            smem_u32(dst)),
        "l"((uint64_t)map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}
// Bounded wait as mbar_wait_bounded, with a short slow path: the waits of the
// issuing warp run once per block of keys between two softmax warps whose code
// fills the instruction cache, and every line of its own that it has to fetch
// again costs more than the instructions in it.
__device__ __forceinline__ bool pk_wait(uint64_t *bar, uint32_t parity, int *err, int code) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = globaltimer_ns();
#pragma unroll 1
    while (!mbar_try_wait(bar, parity))
        if (globaltimer_ns() - t0 > 1000000000ull) {
            if (err) atomicCAS(err, 0, code);
            return false;
        }
    return true;
}
__device__ __forceinline__ uint64_t pk_join(uint32_t lo, uint32_t hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
    return d;
}
__device__ __forceinline__ void pk_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void pk_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void pk_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pk_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// One lane of a converged warp: unlike `lane == 0` it keeps the operands of what
// follows in uniform registers, where tcgen05.mma takes them (with a plain lane
// test a tile's 16 instructions took 1800 cycles to issue, more than they run).
__device__ __forceinline__ bool pk_elect() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
    return p != 0;
}
// D[tmem] (+)= A[smem] B[smem]
__device__ __forceinline__ void pk_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
// D[tmem] (+)= A[tmem] B[smem]
__device__ __forceinline__ void pk_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
#define WK_R32(v, o)                                                                                                 \
    "=r"(v[o]), "=r"(v[o + 1]), "=r"(v[o + 2]), "=r"(v[o + 3]), "=r"(v[o + 4]), "=r"(v[o + 5]), "=r"(v[o + 6]),       \
        "=r"(v[o + 7]), "=r"(v[o + 8]), "=r"(v[o + 9]), "=r"(v[o + 10]), "=r"(v[o + 11]), "=r"(v[o + 12]),            \
        "=r"(v[o + 13]), "=r"(v[o + 14]), "=r"(v[o + 15]), "=r"(v[o + 16]), "=r"(v[o + 17]), "=r"(v[o + 18]),         \
        "=r"(v[o + 19]), "=r"(v[o + 20]), "=r"(v[o + 21]), "=r"(v[o + 22]), "=r"(v[o + 23]), "=r"(v[o + 24]),         \
        "=r"(v[o + 25]), "=r"(v[o + 26]), "=r"(v[o + 27]), "=r"(v[o + 28]), "=r"(v[o + 29]), "=r"(v[o + 30]),         \
        "=r"(v[o + 31])
#define WK_I32(v, o)                                                                                                 \
    "r"(v[o]), "r"(v[o + 1]), "r"(v[o + 2]), "r"(v[o + 3]), "r"(v[o + 4]), "r"(v[o + 5]), "r"(v[o + 6]),              \
        "r"(v[o + 7]), "r"(v[o + 8]), "r"(v[o + 9]), "r"(v[o + 10]), "r"(v[o + 11]), "r"(v[o + 12]),                  \
        "r"(v[o + 13]), "r"(v[o + 14]), "r"(v[o + 15]), "r"(v[o + 16]), "r"(v[o + 17]), "r"(v[o + 18]),               \
        "r"(v[o + 19]), "r"(v[o + 20]), "r"(v[o + 21]), "r"(v[o + 22]), "r"(v[o + 23]), "r"(v[o + 24]),               \
        "r"(v[o + 25]), "r"(v[o + 26]), "r"(v[o + 27]), "r"(v[o + 28]), "r"(v[o + 29]), "r"(v[o + 30]),               \
        "r"(v[o + 31])
// 32 columns of this warp's 32 TMEM lanes, one lane per thread (no wait)
__device__ __forceinline__ void pk_ld(uint32_t taddr, uint32_t *v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : WK_R32(v, 0)
        : "r"(taddr));
}
__device__ __forceinline__ void pk_st(uint32_t taddr, const uint32_t *v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        WK_I32(v, 0)
        : "memory");
}
__device__ __forceinline__ void pk_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pk_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// two fp32 values per instruction
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pk_pair(float lo, float hi) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ f32x2 pk_pair(uint32_t lo, uint32_t hi) {
    return pk_pair(__uint_as_float(lo), __uint_as_float(hi));
}
__device__ __forceinline__ float2 pk_unpair(f32x2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ f32x2 pk_fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f32x2 pk_add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// the largest of three (of those that are not NaN)
__device__ __forceinline__ float pk_max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// shared-memory descriptors, 128-byte swizzle: K-major rows of 128 bytes (8-row
// groups 1024 bytes apart), and MN-major (the contraction runs over the rows;
// 64-element column blocks `lbo` bytes apart)
__device__ __forceinline__ uint64_t pk_desc(uint32_t saddr, uint32_t lbo) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)(lbo >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
           (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
template <typename T> struct PkType {
    static constexpr uint32_t fmt = 0;                  // kind::f16 operand format: f16
    static constexpr uint32_t exp_one = 0x04000400u;    // one unit of the exponent field, both halves
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<uint32_t *>(&h);
    }
};
template <> struct PkType<__nv_bfloat16> {
    static constexpr uint32_t fmt = 1;
    static constexpr uint32_t exp_one = 0x00800080u;
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<uint32_t *>(&h);
    }
};

struct PkArgs {
    void *out;
    long out_rs;
    const int *q_starts, *k_starts;
    int n, q_rows, k_rows, G, GT, chunks;  // heads per K/V head, heads per tile, tiles of heads per K/V head
    int PT;                                // positions per tile
    float scale_log2, shift;               // shift: the bias of P in units of the scores
    int vec;  // out is 16-byte aligned and strided
    int split;  // CTAs of a cluster, which share a unit's keys
    int reach;  // sequences of up to so many keys are left to the short kernel (-1: none)
    int *err;
};

__device__ __forceinline__ void pk_cluster_sync() {
    asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t pk_peer(const void *p, uint32_t rank) {  // p in the shared memory of CTA `rank`
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ float pk_ld_peer(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 pk_ld_peer4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

template <typename T, int D>
__global__ void __launch_bounds__(kPkThreads, 1)
    attn_packed_kernel(const __grid_constant__ PkMaps maps, const PkArgs a) {
    using L = PkLayout<D>;
    constexpr int ST = L::kStages;
    extern __shared__ __align__(1024) uint8_t pk_smem[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)pk_smem + 1023) & ~(uintptr_t)1023);
    PkBars<D> *B = reinterpret_cast<PkBars<D> *>(smem + L::kBars);
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // known to be the same in the whole warp
    if (warp == 9) {  // the loading warp, which waits for nobody before its first loads
        if (lane == 0) {
            mbar_init(&B->q_full, 1);
            for (int i = 0; i < ST; ++i) {
                mbar_init(&B->kv_full[i], 1);
                mbar_init(&B->kv_empty[i], 1);
            }
            for (int i = 0; i < 2; ++i) {
                mbar_init(&B->s_full[i], 1);
                mbar_init(&B->p_half[i], 128);
                mbar_init(&B->p_full[i], 128);
                mbar_init(&B->o_full[i], 1);
            }
            for (int i = 0; i < 4; ++i) {
                mbar_init(&B->v_raw[i], 1);
                mbar_init(&B->v_clean[i], 64);
            }
            mbar_fence_init();
        } else if (lane < 4) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(lane == 1 ? &maps.q : lane == 2 ? &maps.k : &maps.v) : "memory");
        }
        __syncwarp();
    } else if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&B->tmem))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        B->unit.valid = 0;
        B->bad = 0;
    }
    if (tid < D) B->bad_key[tid] = 0x7fffffff;
    pk_fence_before();
    pdl_wait();
    pdl_trigger();
    // ---- this CTA's unit: the idx-th from the end, so that the longest rows of a long prompt start first
    const int idx = blockIdx.z * kPkGridY + blockIdx.y;
    const int rank = a.split == 1 ? 0 : blockIdx.x % a.split, hb = a.split == 1 ? blockIdx.x : blockIdx.x / a.split;
    const int kvh = a.chunks == 1 ? hb : hb / a.chunks, chunk = a.chunks == 1 ? 0 : hb % a.chunks;
    const int PT = a.PT;
    PkUnit unit = {0, 0, 0, 0, 0, 0};
    // sequence i, counted from the end, and its units
    auto look = [&](int i, int &units) -> PkUnit {
        PkUnit s = {0, 0, 0, 0, 0, 0};
        units = 0;
        if (i < a.n) {
            i = a.n - 1 - i;
            const int q0 = a.q_starts[i], q1 = a.q_starts[i + 1], k0 = a.k_starts[i], k1 = a.k_starts[i + 1];
            s.q0 = min(max(q0, 0), a.q_rows);
            s.ql = min(max(q1, s.q0), a.q_rows) - s.q0;
            s.k0 = min(max(k0, 0), a.k_rows);
            s.kl = min(max(k1, s.k0), a.k_rows) - s.k0;
            units = s.kl > a.reach ? (s.ql + 2 * PT - 1) / (2 * PT) : 0;
        }
        return s;
    };
    if (a.n <= 32) {
        // the loading warp for itself, warp 0 for the others
        if (warp == 9 || warp == 0) {
            int units;
            const PkUnit s = look(lane, units);
            int in = units;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, in, o);
                if (lane >= o) in += v;
            }
            const uint32_t who = __ballot_sync(0xffffffffu, idx >= in - units && idx < in);
            if (who) {
                const int from = __ffs(who) - 1;
                unit.valid = 1;
                unit.q0 = __shfl_sync(0xffffffffu, s.q0, from);
                unit.ql = __shfl_sync(0xffffffffu, s.ql, from);
                unit.k0 = __shfl_sync(0xffffffffu, s.k0, from);
                unit.kl = __shfl_sync(0xffffffffu, s.kl, from);
                unit.j0 = (__shfl_sync(0xffffffffu, in, from) - 1 - idx) * 2 * PT;
                if (warp == 0 && lane == 0) B->unit = unit;
            }
        }
        if (warp == 9)
            asm volatile("bar.arrive 2, %0;" ::"n"(kPkThreads) : "memory");
        else
            asm volatile("bar.sync 2, %0;" ::"n"(kPkThreads) : "memory");
    } else {
        int before = 0;
        for (int i0 = 0; i0 < a.n; i0 += kPkThreads) {
            int units;
            PkUnit s = look(i0 + tid, units);
            int in = units;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, in, o);
                if (lane >= o) in += v;
            }
            __syncthreads();
            if (lane == 31) B->units[warp] = in;
            __syncthreads();
            int first = before + in - units;
#pragma unroll
            for (int w = 0; w < kPkThreads / 32; ++w) {
                if (w < warp) first += B->units[w];
                before += B->units[w];
            }
            if (idx >= first && idx < first + units) {
                s.valid = 1;
                s.j0 = (units - 1 - (idx - first)) * 2 * PT;
                B->unit = s;
            }
            if (idx < before) break;
        }
        __syncthreads();
    }
    if (warp != 9 || a.n > 32) unit = B->unit;
    pk_fence_after();
    const uint32_t tmem = B->tmem;
    bool ok = true;
    if (unit.valid) {
        const int q0 = unit.q0, ql = unit.ql;
        const int j0 = unit.j0;  // first query of the unit
        const int head0 = kvh * a.G + chunk * a.GT;
        // The unit's last query sees `all` blocks of keys; this CTA's share of them starts at
        // block `skip`, and from here on keys count from there.
        const int all = max(0, (unit.kl - ql + min(j0 + 2 * PT, ql) - 1 + kPkKeys) / kPkKeys);
        const int share = a.split == 1 ? all : (all + a.split - 1) / a.split, skip = rank * share;
        const int k0 = unit.k0 + skip * kPkKeys, kl = unit.kl - skip * kPkKeys;
        const int shift = kl - ql;  // query j sees keys 0 .. shift + j
        // blocks of keys that each tile sees (0: none), and the first that some row of the unit sees in part
        auto blocks = [&](int t) -> int {
            const int f = j0 + t * PT;
            if (f >= ql) return 0;
            const int last = shift + min(f + PT, ql) - 1;  // the last key that the tile sees
            return last < 0 ? 0 : min(last / kPkKeys + 1, share);
        };
        const int n0 = blocks(0), n1 = blocks(1), nb = max(n0, n1);
        const int part = max(0, (shift + j0 + 1) / kPkKeys);  // blocks below this are seen whole by every row
        // registers: 256 softmax threads x 216 + 128 x 72 = the launch's 384 x 168
        if (warp >= 8) {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
            if (warp == 9) {
                if (nb > 0 && pk_elect()) {
                    const uint32_t qbytes = (uint32_t)(PT * a.GT) * D * 2;
                    auto load_q = [&](int t) {
                        for (int b = 0; b < D / 64; ++b)
                            pk_tma3(smem + L::kQ + t * L::kTile + b * 16384, &maps.q, 64 * b, head0, q0 + j0 + t * PT,
                                    &B->q_full);
                    };
                    mbar_expect_tx(&B->q_full, n0 > 0 && n1 > 0 ? 2 * qbytes : qbytes);
                    if (n0 > 0) load_q(0);
                    auto raw = [&](int i) -> uint64_t * {
                        return (i & 1) && (i >> 1) >= part ? &B->v_raw[((i >> 1) - part) & 3] : nullptr;
                    };
                    int issued = 0;
                    for (int i = 0; i < 2 * nb; ++i) {
                        const int s = i % ST;
                        if (i >= ST && !pk_wait(&B->kv_empty[s], ((i / ST) - 1) & 1, a.err, 50)) {
                            ok = false;
                            break;
                        }
                        uint64_t *bar = &B->kv_full[s];
                        if (raw(i)) {  // lands on a barrier of its own; the ring's only keeps step
                            pk_arrive(bar);
                            bar = raw(i);
                        }
                        mbar_expect_tx(bar, L::kTile);
                        const CUtensorMap *m = (i & 1) ? &maps.v : &maps.k;
                        for (int b = 0; b < D / 64; ++b)
                            pk_tma3(smem + L::kRing + (size_t)s * L::kTile + b * 16384, m, 64 * b, kvh,
                                    k0 + (i >> 1) * kPkKeys, bar);
                        ++issued;
                        if (i == 0 && n1 > 0) load_q(1);
                    }
                    if (!ok)  // no copy of this CTA may land after it has left
                        for (int i = max(0, issued - ST); i < issued; ++i) {
                            if (raw(i))
                                pk_wait(raw(i), (((i >> 1) - part) >> 2) & 1, a.err, 51);
                            else
                                pk_wait(&B->kv_full[i % ST], (i / ST) & 1, a.err, 51);
                        }
                }
            } else if (warp == 8) {
                if (nb > 0 && pk_elect()) {
                    constexpr uint32_t fmt = (1u << 4) | (PkType<T>::fmt << 7) | (PkType<T>::fmt << 10) | (8u << 24);
                    constexpr uint32_t id_qk = fmt | (uint32_t)(kPkKeys >> 3) << 17;
                    constexpr uint32_t id_pv = fmt | (1u << 16) | (uint32_t)(D >> 3) << 17;  // B (V) MN-major
                    const uint32_t ring = smem_u32(smem + L::kRing), qs = smem_u32(smem + L::kQ);
                    // the halves of a descriptor: the upper is constant, the lower the address
                    const uint32_t q_lo = (uint32_t)pk_desc(qs, 16), ring_lo = (uint32_t)pk_desc(ring, 16);
                    constexpr uint32_t hi = (uint32_t)(1024 >> 4) | 1u << 14 | 2u << 29;
                    constexpr uint32_t mn = (uint32_t)(16384 >> 4) << 16;  // V: leading offset of the next 64 dimensions
                    constexpr uint32_t step = L::kTile >> 4;
                    auto qk = [&](int t, int stage) {
                        const uint32_t kb = ring_lo + stage * step, qb = q_lo + t * step;
#pragma unroll
                        for (int kk = 0; kk < D / 16; ++kk) {
                            const uint32_t o = ((kk >> 2) * 16384 + (kk & 3) * 32) >> 4;
                            pk_mma_ss(tmem + t * 128, pk_join(qb + o, hi), pk_join(kb + o, hi), id_qk, kk != 0);
                        }
                        pk_commit(&B->s_full[t]);
                    };
                    auto pv = [&](int t, int stage, int half, uint32_t acc) {
                        const uint32_t vb = (ring_lo & 0xffffu) + stage * step + mn + half * (4 * 2048 >> 4);
                        const uint32_t pb = tmem + t * 128 + 32 * half;
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            pk_mma_ts(tmem + 256 + t * 128, pb + 8 * kk, pk_join(vb + kk * (2048 >> 4), hi), id_pv, acc | kk);
                    };
                    // A wait costs 150 to 200 cycles even when its barrier is done (it queues behind
                    // the softmax warps' exponentials), so the waits for K and V come while the first
                    // tile's softmax still runs, and the commits that nobody waits for come last.
                    int stage = 0;
                    uint32_t phase = 0;
                    auto next = [&]() {
                        if (++stage == ST) {
                            stage = 0;
                            phase ^= 1;
                        }
                    };
                    ok = pk_wait(&B->q_full, 0, a.err, 53) && pk_wait(&B->kv_full[0], 0, a.err, 52);
                    if (ok) {
                        pk_fence_after();
                        if (n0 > 0) qk(0, 0);
                        if (n1 > 0) qk(1, 0);
                        pk_commit(&B->kv_empty[0]);
                    }
                    next();
#pragma unroll 1
                    for (int j = 0; j < nb && ok; ++j) {
                        const int vs = stage;
                        ok = pk_wait(&B->kv_full[vs], phase, a.err, 52);
                        if (j >= part) ok = ok && pk_wait(&B->v_clean[(j - part) & 3], ((j - part) >> 2) & 1, a.err, 54);
                        next();
                        const int ks = stage;
                        if (j + 1 < nb) ok = ok && pk_wait(&B->kv_full[ks], phase, a.err, 52);
                        next();
#pragma unroll 1
                        for (int t = 0; t < 2; ++t) {
                            const int nt = t ? n1 : n0;
                            if (j < nt) {
                                ok = ok && pk_wait(&B->p_half[t], j & 1, a.err, 55);
                                if (!ok) break;
                                pk_fence_after();
                                pv(t, vs, 0, j);
                                ok = pk_wait(&B->p_full[t], j & 1, a.err, 60);
                                if (!ok) break;
                                pk_fence_after();
                                pv(t, vs, 1, 1);
                                if (j + 1 == nt) pk_commit(&B->o_full[t]);
                            }
                            if (j + 1 < nt) qk(t, ks);
                        }
                        if (ok) {
                            pk_commit(&B->kv_empty[vs]);
                            if (j + 1 < nb) pk_commit(&B->kv_empty[ks]);
                        }
                    }
                }
            } else {
                // ---- V of the blocks that are seen in part
                const int ct = tid - 320;  // 0..63
                for (int j = part; j < nb && ok; ++j) {
                    const int s = (2 * j + 1) % ST, c = j - part;
                    if (!pk_wait(&B->v_raw[c & 3], (c >> 2) & 1, a.err, 56)) {
                        ok = false;
                        break;
                    }
                    uint8_t *vb = smem + L::kRing + (size_t)s * L::kTile;
                    const int live = min(kPkKeys, kl - j * kPkKeys);
                    // 16-byte chunks: chunk c of key row r lies at place c ^ (r & 7) of its 128 bytes
                    constexpr uint32_t e = PkType<T>::exp_one;
                    uint4 *vq = reinterpret_cast<uint4 *>(vb) + ct;
#pragma unroll 1
                    for (int q = 0; q < kPkKeys * D / 8; q += 8 * 64) {
                        uint4 u[8];
                        uint32_t hit = 0;
#pragma unroll
                        for (int x = 0; x < 8; ++x) u[x] = vq[q + 64 * x];
#pragma unroll
                        for (int x = 0; x < 8; ++x) {
                            const int r = ((ct + q + 64 * x) >> 3) & 127;
                            if (r >= live)
                                vq[q + 64 * x] = make_uint4(0, 0, 0, 0);
                            else
                                hit |= ((u[x].x & 0x7fff7fffu) + e) | ((u[x].y & 0x7fff7fffu) + e) |
                                       ((u[x].z & 0x7fff7fffu) + e) | ((u[x].w & 0x7fff7fffu) + e);
                        }
                        if (hit & 0x80008000u) {  // rare
                            unsigned short *v = reinterpret_cast<unsigned short *>(vq + q);
#pragma unroll 1
                            for (int y = 0; y < 64; ++y) {
                                const int x = y >> 3, c = ct + q + 64 * x, r = (c >> 3) & 127;
                                unsigned short *w = v + 64 * 8 * x + (y & 7);
                                if (r < live && ((*w & 0x7fffu) + (e & 0xffffu)) & 0x8000u) {
                                    *w = 0;
                                    atomicMin(&B->bad_key[(c >> 10) * 64 + ((c & 7) ^ (r & 7)) * 8 + (y & 7)],
                                              j * kPkKeys + r);
                                    B->bad = 1;
                                }
                            }
                        }
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    pk_arrive(&B->v_clean[c & 3]);
                }
            }
        } else {
            asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
            // ---- softmax: thread = row of tile t
            const int t = warp >> 2, row = tid & 127;
            const int nt = t ? n1 : n0;
            const int jq = j0 + t * PT + row / a.GT;  // query of this row
            const int lim = shift + jq;               // last key that it sees
            const int lim0 = shift + j0 + t * PT;     // of the tile's first row
            const uint32_t lanes = (uint32_t)(warp & 3) << 21;
            const uint32_t s_t = tmem + t * 128 + lanes, o_t = tmem + 256 + t * 128 + lanes;
            float m = -INFINITY, l = 0.f;  // m: what P is relative to, a maximum less the shift for its bias
            for (int j = 0; j < nt; ++j) {
                // (the warp leaves as one: what follows is warp-wide)
                if (!__all_sync(0xffffffffu, pk_wait(&B->s_full[t], j & 1, a.err, 57))) {
                    ok = false;
                    break;
                }
                pk_fence_after();
                uint32_t sv[128];
#pragma unroll
                for (int c = 0; c < 4; ++c) pk_ld(s_t + 32 * c, sv + 32 * c);
                pk_wait_ld();
                if (j * kPkKeys + kPkKeys - 1 > lim0) {
                    const int seen = lim - j * kPkKeys;  // keys of the block up to this one
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const int s = seen - 32 * w;
                        const uint32_t bits = s >= 31 ? 0xffffffffu : s < 0 ? 0u : (2u << s) - 1u;
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (!(bits >> i & 1u)) sv[32 * w + i] = 0xff800000u;
                    }
                }
                // exponentials of keys 64 c .. 64 c + 63, their sum and P; FIND: the maximum of the
                // block's 128 scores on the way (it uses another pipe than the exponentials)
                const f32x2 scale2 = pk_pair(a.scale_log2, a.scale_log2);
                float mx[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) mx[e] = __uint_as_float(sv[e]);
                auto half = [&](int c, bool find, float m, f32x2(&sum)[2], uint32_t(&pv)[32]) {
                    const float base = m == -INFINITY ? 0.f : __fmul_rd(-m, a.scale_log2);
                    const f32x2 base2 = pk_pair(base, base);
                    sum[0] = sum[1] = 0;
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const f32x2 x = pk_fma2(pk_pair(sv[64 * c + 2 * i], sv[64 * c + 2 * i + 1]), scale2, base2);
                        float2 u = pk_unpair(x);
                        u.x = pk_ex2(u.x);
                        u.y = pk_ex2(u.y);
                        if (find) {
                            float &p = mx[(2 * i) & 3], &r = mx[(2 * i + 1) & 3];
                            p = pk_max3(p, __uint_as_float(sv[4 * i]), __uint_as_float(sv[4 * i + 1]));
                            r = pk_max3(r, __uint_as_float(sv[4 * i + 2]), __uint_as_float(sv[4 * i + 3]));
                        }
                        sum[i & 1] = pk_add2(sum[i & 1], pk_pair(u.x, u.y));
                        pv[i] = PkType<T>::pack(u.x, u.y);
                    }
                };
                // The first half is computed with the maximum so far while this block's is
                // found, and again in the rare case that the maximum moves.  (Before the first
                // block, the maximum of 16 keys is near enough: code that runs once per unit
                // costs its way through the instruction cache.)
                f32x2 sum[2];
                uint32_t pv[32];
                if (j == 0) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) m = fmaxf(m, __uint_as_float(sv[i]));
                    m = __fsub_ru(m, a.shift);
                }
                half(0, true, m, sum, pv);
                const float mb = __fsub_ru(pk_max3(pk_max3(mx[0], mx[1], mx[2]), mx[3], mx[3]), a.shift);
                const bool move = (mb - m) * a.scale_log2 > PkWeight<T>::lead || (m == -INFINITY && mb > m);
                if (__any_sync(0xffffffffu, move)) {
                    const float mn = move ? mb : m;
                    const float f = mn == m || m == -INFINITY ? 1.f : pk_ex2((m - mn) * a.scale_log2);
                    m = mn;
                    l *= f;
                    if (j > 0) {  // the products so far are complete: S of this block was issued after them
#pragma unroll
                        for (int c = 0; c < D / 32; ++c) {
                            uint32_t ov[32];
                            pk_ld(o_t + 32 * c, ov);
                            pk_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * f);
                            pk_st(o_t + 32 * c, ov);
                        }
                    }
                    half(0, false, m, sum, pv);
                }
                // P goes to the tensor cores in two halves, the first while the second is computed
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    if (c) half(1, false, m, sum, pv);
                    const float2 u = pk_unpair(pk_add2(sum[0], sum[1]));
                    l += u.x + u.y;
                    pk_st(s_t + 32 * c, pv);
                    pk_wait_st();
                    pk_fence_before();
                    pk_arrive(c ? &B->p_full[t] : &B->p_half[t]);
                }
            }
            // ---- epilogue
            if (nt > 0 && ok && !__all_sync(0xffffffffu, pk_wait(&B->o_full[t], 0, a.err, 58))) ok = false;
            pk_fence_after();
            // what the clearing warps noted of this tile's blocks
            if (nt > part && ok) pk_wait(&B->v_clean[(nt - 1 - part) & 3], ((nt - 1 - part) >> 2) & 1, a.err, 59);
            const bool bad = nt > 0 && B->bad;
            const float inv = l > 0.f || l != l ? 1.f / l : 0.f;  // a row that sees nothing has O = 0 and l = 0
            // 32 values of this row from TMEM
            auto load_o = [&](int c, uint32_t(&ov)[32]) {
                if (nt > 0) {
                    pk_ld(o_t + 32 * c, ov);
                    pk_wait_ld();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) ov[i] = 0;
                }
                if (bad) {
                    const int4 *key = reinterpret_cast<const int4 *>(&B->bad_key[32 * c]);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int4 k = key[i];
                        ov[4 * i] = k.x <= lim ? 0x7fc00000u : ov[4 * i];
                        ov[4 * i + 1] = k.y <= lim ? 0x7fc00000u : ov[4 * i + 1];
                        ov[4 * i + 2] = k.z <= lim ? 0x7fc00000u : ov[4 * i + 2];
                        ov[4 * i + 3] = k.w <= lim ? 0x7fc00000u : ov[4 * i + 3];
                    }
                }
            };
            // Where row x of tile s goes (null: nowhere).  (The unit is read again from shared
            // memory, which keeps the loop over the blocks free of what only the end needs.)
            auto row_out = [&](int s, int x) -> T * {
                const PkUnit &un = B->unit;
                const int j = un.j0 + s * PT + x / a.GT, h = chunk * a.GT + x % a.GT;
                if (x >= PT * a.GT || j >= un.ql || h >= a.G || !ok) return nullptr;
                return reinterpret_cast<T *>(a.out) + (long)(un.q0 + j) * a.out_rs + (long)(kvh * a.G + h) * D;
            };
            if (a.split == 1) {
                // The warp's rows through the part of the Q tile that they came from (all products
                // that read it are complete), so that a row is written by consecutive lanes.
                constexpr int C = D / 8;  // 16-byte chunks per row, chunk c of row r at place c ^ (r & 7)
                uint4 *buf = reinterpret_cast<uint4 *>(smem + L::kQ + t * L::kTile) + (warp & 3) * 32 * C;
                const T *own = row_out(t, row);  // the row in this lane's registers
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t ov[32], w[16];
                    load_o(c, ov);
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        w[i] = PkType<T>::pack(__uint_as_float(ov[2 * i]) * inv, __uint_as_float(ov[2 * i + 1]) * inv);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        buf[lane * C + ((4 * c + i) ^ (lane & 7))] =
                            make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                }
                __syncwarp();
                const int c = lane % C;  // this lane's chunk of each row that it writes
#pragma unroll 2
                for (int x = 0; x < C; ++x) {
                    const int r = x * (32 / C) + lane / C;
                    T *o = reinterpret_cast<T *>(__shfl_sync(0xffffffffu, (unsigned long long)own, r));
                    const uint4 v = buf[r * C + (c ^ (r & 7))];
                    if (o && a.vec) {
                        reinterpret_cast<uint4 *>(o)[c] = v;
                    } else if (o) {
                        unsigned short *e = reinterpret_cast<unsigned short *>(o) + 8 * c;
                        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            e[2 * i] = (unsigned short)w[i];
                            e[2 * i + 1] = (unsigned short)(w[i] >> 16);
                        }
                    }
                }
            } else {
                // O as it stands into the ring, which the products of both tiles have left (16-byte
                // chunk c of row r at place c ^ (r & 7)), the maxima and sums into the Q tiles' place
                constexpr int C = D / 4;
                asm volatile("bar.sync 1, 256;" ::: "memory");
                float4 *buf = reinterpret_cast<float4 *>(smem + L::kRing) + (t * 128 + row) * C;
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t ov[32];
                    load_o(c, ov);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        buf[(8 * c + i) ^ (row & 7)] =
                            make_float4(__uint_as_float(ov[4 * i]), __uint_as_float(ov[4 * i + 1]),
                                        __uint_as_float(ov[4 * i + 2]), __uint_as_float(ov[4 * i + 3]));
                }
                float *part_m = reinterpret_cast<float *>(smem + L::kQ), *part_l = part_m + 256;
                part_m[tid] = m * a.scale_log2;
                part_l[tid] = l;
                pk_cluster_sync();
                // this CTA joins and writes its share of the rows, D / 4 lanes to a row
                const int rows = (256 + a.split - 1) / a.split, r1 = min(256, (rank + 1) * rows);
                for (int r = rank * rows + tid / C; r < r1; r += 256 / C) {
                    T *o = row_out(r >> 7, r & 127);
                    if (!o) continue;
                    const int c = tid % C;
                    float top = -INFINITY;
                    for (int x = 0; x < a.split; ++x) top = fmaxf(top, pk_ld_peer(pk_peer(&part_m[r], x)));
                    float sum = 0.f;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    for (int x = 0; x < a.split; ++x) {
                        const float mx = pk_ld_peer(pk_peer(&part_m[r], x)), lx = pk_ld_peer(pk_peer(&part_l[r], x));
                        const float4 ox = pk_ld_peer4(
                            pk_peer(reinterpret_cast<float4 *>(smem + L::kRing) + r * C + (c ^ (r & 7)), x));
                        const float f = mx == -INFINITY ? (lx != lx ? 1.f : 0.f) : pk_ex2(mx - top);
                        sum += lx * f;
                        v.x += ox.x * f;
                        v.y += ox.y * f;
                        v.z += ox.z * f;
                        v.w += ox.w * f;
                    }
                    const float is = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
                    const uint32_t w0 = PkType<T>::pack(v.x * is, v.y * is), w1 = PkType<T>::pack(v.z * is, v.w * is);
                    if (a.vec) {
                        reinterpret_cast<uint2 *>(o)[c] = make_uint2(w0, w1);
                    } else {
                        unsigned short *e = reinterpret_cast<unsigned short *>(o) + 4 * c;
                        e[0] = (unsigned short)w0;
                        e[1] = (unsigned short)(w0 >> 16);
                        e[2] = (unsigned short)w1;
                        e[3] = (unsigned short)(w1 >> 16);
                    }
                }
            }
        }
        if (a.split > 1) {
            __syncwarp();
            if (warp >= 8) pk_cluster_sync();  // the softmax warps' first
            pk_cluster_sync();                 // no CTA leaves while its part is read
        }
    }
    pk_fence_before();
    __syncthreads();
    pk_fence_after();
    if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// 3-D map over [rows][heads][D] 16-bit values with boxes of box_rows x box_heads x 64.
bool pk_map(CUtensorMap *m, const void *base, int dtype, int D, int heads, int rows, long rs, int box_heads,
            int box_rows) {
    return encode_map_3d(m, base, dtype == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                         D, heads, rows, 2 * (uint64_t)D, 2 * (uint64_t)rs, 64, box_heads, box_rows,
                         CU_TENSOR_MAP_SWIZZLE_128B);
}

// Sets the tcgen05 kernel up on the current device.  *fits: it has the registers that its split
// counts on; where a compiler gave it others, the split would wait for registers that the launch
// does not have, and the other kernels serve.
template <typename T, int D> cudaError_t ready_packed(bool *fits) {
    constexpr size_t smem = PkLayout<D>::kBars + sizeof(PkBars<D>) + 1024;
    static_assert(smem <= 232448, "shared memory of a CTA");
    auto kern = attn_packed_kernel<T, D>;
    static int configured = -1;  // the device that the kernel is set up for
    static bool as_split = false;
    if (configured != g_rt.device) {
        cudaFuncAttributes fa;
        cudaError_t e = cudaFuncGetAttributes(&fa, kern);
        if (e != cudaSuccess) return e;
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
        as_split = fa.numRegs == kPkRegs;
        configured = g_rt.device;
    }
    *fits = as_split && g_rt.tc_attn;
    return cudaSuccess;
}

template <typename T, int D> cudaError_t launch_packed(const PackedArgs &p, const PkMaps &maps, int GT, cudaStream_t s) {
    constexpr size_t smem = PkLayout<D>::kBars + sizeof(PkBars<D>) + 1024;
    auto kern = attn_packed_kernel<T, D>;
    PkArgs a;
    a.out = p.out;
    a.out_rs = p.out_rs;
    a.q_starts = p.q_starts;
    a.k_starts = p.k_starts;
    a.n = p.n;
    a.q_rows = p.q_rows;
    a.k_rows = p.k_rows;
    a.G = p.heads / p.kv_heads;
    a.GT = GT;
    a.chunks = (a.G + GT - 1) / GT;
    a.PT = 128 / GT;
    a.scale_log2 = p.scale * 1.4426950408889634f;
    a.shift = PkWeight<T>::bias / a.scale_log2;
    a.vec = ((uintptr_t)p.out % 16) == 0 && p.out_rs % 8 == 0;
    a.reach = p.reach;
    a.err = g_rt.d_error;
    const int PT = 128 / GT;
    // units: ceil(length / (2 PT)) per sequence
    const int n = p.longer;  // that are this kernel's
    const long long most = n == 1 ? (p.q_rows + 2ll * PT - 1) / (2 * PT) : (long long)p.q_rows / (2 * PT) + n;
    const long long units = most < p.q_rows ? most : p.q_rows;
    const long long ctas = units * p.kv_heads * a.chunks;
    const long long z = (units + kPkGridY - 1) / kPkGridY;
    if ((long long)p.kv_heads * a.chunks * 8 > 0x7fffffffll || z > 65535) return cudaErrorInvalidConfiguration;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kPkThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = g_rt.pdl ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    // Few units and long sequences: a cluster to each, where all run at once and it saves more
    // blocks of keys (of the mean length) than its join takes: 11 us with 2 or 3 CTAs, 8 us
    // with more, heads of 64 7 and 5 us, 3 us where a unit has a row or two, a block taking
    // 1.6.  8 heads of 128 over 1, us without / with 2 / 4 / 8 CTAs to a unit:
    //   512 rows  13.8 / 21.7 / 16.5 / 30.0 (16 clusters of 8 do not fit)   500 behind 4000  67 / 48 / 30 / 40
    //   1024      20.6 / 25.2 / 18.3 / -     2048  34.1 / 32.6 / - / -      2000 behind 14000  216 / 126 / - / -
    static int at_once[9], at_once_on = -1;  // clusters of a size that run at once, on which device
    if (at_once_on != g_rt.device) {
        for (int c = 2; c <= 8; ++c) {
            cfg.gridDim = dim3(c);
            attr[1].val.clusterDim.x = c;
            cfg.numAttrs = 2;
            const cudaError_t e = cudaOccupancyMaxActiveClusters(&at_once[c], kern, &cfg);
            if (e != cudaSuccess) return e;
        }
        at_once_on = g_rt.device;
    }
    const double blocks = (double)p.k_rows / ((double)kPkKeys * n);
    long long split = blocks / 2 < g_rt.num_sms / ctas ? (long long)(blocks / 2) : g_rt.num_sms / ctas;
    if (split > 8) split = 8;
    // (of one sequence the units are exact; of several they are fewer than `units`, which leaves room)
    while (split > 1 && at_once[split] < (n == 1 ? ctas : 1)) --split;
    const double full = (double)p.q_rows / ((double)n * 2 * PT);  // how full units are, on average
    const double join = 2 + (full < 1 ? full : 1) * ((D == 64 ? 1 : 3) + (split < 4 ? D / 64 : 0));  // in blocks
    const double longer = n > 2 ? 1.5 : 1;  // of several, the longest ends last
    if (blocks * longer * (split - 1) < split * join) split = 1;
    a.split = split < 2 ? 1 : (int)split;
    cfg.gridDim = dim3(p.kv_heads * a.chunks * a.split, (unsigned)(units < kPkGridY ? units : kPkGridY), (unsigned)z);
    attr[1].val.clusterDim.x = a.split;
    cfg.numAttrs = a.split > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, maps, a);
}

template <typename T, int D> cudaError_t launch_short(const PackedArgs &a, int units, cudaStream_t s) {
    auto kern = attn_packed_short_kernel<T, D>;
    static int configured = -1;
    if (configured != g_rt.device) {
        const cudaError_t e =
            cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, ShLayout<D>::kSmem);
        if (e != cudaSuccess) return e;
        configured = g_rt.device;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.kv_heads, units);
    cfg.blockDim = dim3(128);
    cfg.dynamicSmemBytes = ShLayout<D>::kSmem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = g_rt.pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, a);
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
    if ((((uintptr_t)out | (uintptr_t)q | (uintptr_t)k | (uintptr_t)v) % 2) ||
        (((uintptr_t)q_starts | (uintptr_t)k_starts) % 4))
        return fail("wk_attention_packed: misaligned argument");
    if (g_rt.device < 0) return fail("wk_attention_packed: cuda_init() has not been called");
    DeviceGuard guard;
    PackedArgs a{out, out_rs, q, k, v, q_rs, k_rs, v_rs, q_starts, k_starts, n, q_rows, k_rows, n_heads, kv_heads,
                 1.0f / sqrtf((float)head_dim), (uintptr_t)out % 4 == 0 && out_rs % 2 == 0, -1, n};
    cudaStream_t s = stream();
    cudaError_t e = cudaSuccess;
    // TMA wants 16-byte aligned bases and strides; what is not goes row by row
    bool by_rows = true;
    const uintptr_t low = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v;
    if (low % 16 == 0 && (q_rs | k_rs | v_rs) % 8 == 0 && k_rows > 0) {
        const int G = n_heads / kv_heads, GT = G < 128 ? G : 128;
        // Short sequences go to the kernel for them.  The host knows room and count only, and idle
        // sequences and room without rows hide a long one; so where all of them may be short but one
        // could be long, both kernels are launched and each takes its own sequences by their lengths.
        // The second launch takes the host 2 us, so up to `alone` keys in all the short kernel serves
        // alone; above `mean`, both take no less than the tcgen05 kernel alone.  us, short kernel /
        // tcgen05 / both, 32 / 8 heads of 128:
        //   1 of 192             9.6 / 10.1         24 of 16     7.4 / 15.0         100 of 16  15.0 / 44.1 / 19.0
        //   1 of 256            11.6 / 10.2         24 of 40    13.0 / 17.3 / 14.9  100 of 40  36.8 / 55.1 / 45.4
        //   512 and 63 of 0     26.8 / 13.9         24 of 60    14.8 / 17.3 / 18.4  400 of 40   144 /  231 /  182
        //   4096 and 63 of 0     452 /  127 /  129  24 of 97    26.6 / 26.3
        // 16 / 4 heads of 64:
        //   1 of 384             9.5 / 10.2         24 of 40     5.5 /  7.4         100 of 40  11.7 / 22.7 / 15.7
        //   1 of 768            17.3 / 16.8         24 of 97    10.1 / 14.0 / 13.4  400 of 97   109 /  175 /  150
        //   4096 and 63 of 0     134 /   59 /   60  24 of 200   16.9 / 20.7
        const int reach = head_dim == 64 ? 512 : 256;
        const int alone = head_dim == 64 ? 640 : 512;
        const int mean = head_dim == 64 ? 112 : 48;
        // base(n) of that kernel, with all rows
        long long units = (long long)q_rows * G / 64 + n;
        if (units > q_rows) units = q_rows;
        const bool can_short = G <= 64 && units <= 65535 && kv_heads <= 65535;
        bool some_short =
            can_short && (n == 1 ? k_rows <= reach * 3 / 4 : k_rows <= alone || k_rows <= (long long)mean * n);
        bool some_long = !some_short || k_rows > alone;
        const int longer = k_rows / (reach + 1);  // key rows are nobody's twice
        a.reach = !some_short ? -1 : some_long ? reach : k_rows;
        a.longer = some_short && longer < n ? longer : n;
        if (some_long) {
            bool fits = false;
            if (dtype == kF16)
                e = head_dim == 64 ? ready_packed<__half, 64>(&fits) : ready_packed<__half, 128>(&fits);
            else
                e = head_dim == 64 ? ready_packed<__nv_bfloat16, 64>(&fits) : ready_packed<__nv_bfloat16, 128>(&fits);
            if (e != cudaSuccess) return fail_cuda("wk_attention_packed", e);
            if (!fits) {  // all are the short kernel's, or go row by row
                some_long = false;
                some_short = can_short;
                a.reach = k_rows;
            }
        }
        if (some_long) {
            PkMaps maps;
            if (!pk_map(&maps.q, q, dtype, head_dim, n_heads, q_rows, q_rs, GT, 128 / GT) ||
                !pk_map(&maps.k, k, dtype, head_dim, kv_heads, k_rows, k_rs, 1, kPkKeys) ||
                !pk_map(&maps.v, v, dtype, head_dim, kv_heads, k_rows, v_rs, 1, kPkKeys))
                return fail("wk_attention_packed: cuTensorMapEncodeTiled failed");
            if (dtype == kF16)
                e = head_dim == 64 ? launch_packed<__half, 64>(a, maps, GT, s)
                                   : launch_packed<__half, 128>(a, maps, GT, s);
            else
                e = head_dim == 64 ? launch_packed<__nv_bfloat16, 64>(a, maps, GT, s)
                                   : launch_packed<__nv_bfloat16, 128>(a, maps, GT, s);
        }
        if (some_short && e == cudaSuccess) {
            if (dtype == kF16)
                e = head_dim == 64 ? launch_short<__half, 64>(a, (int)units, s)
                                   : launch_short<__half, 128>(a, (int)units, s);
            else
                e = head_dim == 64 ? launch_short<__nv_bfloat16, 64>(a, (int)units, s)
                                   : launch_short<__nv_bfloat16, 128>(a, (int)units, s);
        }
        by_rows = !some_long && !some_short;
    }
    if (by_rows) {
        if (dtype == kF16)
            e = head_dim == 64 ? launch_rows<__half, 64>(a, s) : launch_rows<__half, 128>(a, s);
        else
            e = head_dim == 64 ? launch_rows<__nv_bfloat16, 64>(a, s) : launch_rows<__nv_bfloat16, 128>(a, s);
    }
    if (e != cudaSuccess) return fail_cuda("wk_attention_packed", e);
    return 0;
}

}  // extern "C"
