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

// The 16-bit types order like their bits below the sign.
template <typename T> struct Kv8Bits {
    static constexpr uint32_t inf = 0x7c00u;
    static __device__ __forceinline__ float value(uint32_t b) { return __half2float(__ushort_as_half((unsigned short)b)); }
};
template <> struct Kv8Bits<__nv_bfloat16> {
    static constexpr uint32_t inf = 0x7f80u;
    static __device__ __forceinline__ float value(uint32_t b) { return __uint_as_float(b << 16); }
};

// Eight 16-bit values from p; VEC: p is 16-byte aligned.
template <bool VEC> __device__ __forceinline__ uint4 load8(const void *p) {
    if (VEC) return *reinterpret_cast<const uint4 *>(p);
    const unsigned short *e = reinterpret_cast<const unsigned short *>(p);
    return make_uint4(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16, e[4] | (uint32_t)e[5] << 16,
                      e[6] | (uint32_t)e[7] << 16);
}
// Two values, times a power of two -> two e4m3 codes, one rounding.
template <typename T> __device__ __forceinline__ uint32_t to_e4m3x2(uint32_t w, float inv) {
    const float lo = Kv8Bits<T>::value(w & 0xffffu), hi = Kv8Bits<T>::value(w >> 16);
    return __nv_cvt_float2_to_fp8x2(make_float2(lo * inv, hi * inv), __NV_SATFINITE, __NV_E4M3);
}

// One CTA per (page that the call writes, K/V head): threads 0..127 take K,
// 128..255 V.  The page's new rows stay in registers, as the 16-bit values that
// they are, between the maximum and the rounding, so each is read once; their
// loads are under way while the block table is read.  Bytes bound long prompts: 9
// of 301 to 2303 tokens, 8 heads of 128, take 13.9 us, 73 % of the copy rate; what is
// left is the chain lengths -> table -> old scale -> rows of each CTA, which six CTAs
// per SM (their register limit) hide in part.  Latency bounds a step of 48 tokens: 7.7 us,
// 3.3 us in a graph.  VEC: rows whose base and stride are multiples of 16 bytes are
// read 16 bytes at a time, others element by element (any alignment of the type).
template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(256, 6) kv8_store_kernel(Kv8Store a) {
    constexpr int kChunks = D / 8;               // 8-element chunks per row
    constexpr int kRows = 128 / kChunks;         // rows per pass of 128 threads
    constexpr int kPasses = kKv8Page / kRows;
    __shared__ int s_found[5];  // sequence, page index, first row, tokens, first offset
    __shared__ uint32_t s_max[8];
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    const int unit = blockIdx.x, head = blockIdx.y;
    if (tid == 0) s_found[0] = -1;
    __syncthreads();
    pdl_wait();
    pdl_trigger();
    // The sequence and page of this CTA.  `add` tokens touch at most add pages, and at most
    // add / 64 + 2; so sequence i has room from base(i) = min(starts, starts / 64 + 2 i) to
    // base(i + 1), and it is found by comparisons alone (a scan over the pages that each touches
    // took 20.6 us instead of 17.8 for 512 sequences of one token, 8 heads of 128; 1092
    // instead of 267 for 8192).
    auto start = [&](int i) -> int { return min(max(a.starts[i], 0), a.rows); };
    auto base = [&](int r, int i) -> int { return (int)min((long)r, r / kKv8Page + 2l * i); };
    int lo = 0, len = a.n;
    while (len > 256) {
        const int st = (len + 255) / 256, i = lo + tid * st;
        const int c = __syncthreads_count(tid * st < len && base(start(i), i) <= unit);
        if (c == 0) return;
        lo += (c - 1) * st;
        len = min(st, len - (c - 1) * st);
    }
    if (tid < len) {
        const int i = lo + tid, r0 = start(i), r1 = start(i + 1), ctx = max(a.ctx[i], 0);
        const int add = r1 - r0, k = unit - base(r0, i);  // its k-th touched page
        const int open = ctx % kKv8Page;
        if (k >= 0 && unit < base(r1, i + 1) && k < (open + add + kKv8Page - 1) / kKv8Page && add > 0) {
            const int before = k ? k * kKv8Page - open : 0;  // tokens before this page
            const int off = k ? 0 : open;
            s_found[0] = i;
            s_found[1] = ctx / kKv8Page + k;
            s_found[2] = r0 + before;
            s_found[3] = min(kKv8Page - off, add - before);
            s_found[4] = off;
        }
    }
    __syncthreads();
    if (s_found[0] < 0 || s_found[1] >= a.max_pages) return;
    const int row0 = s_found[2], m = s_found[3], off = s_found[4];
    const int kv = tid >> 7, t = tid & 127;
    const int c = t % kChunks, r = t / kChunks;
    const long rs = kv ? a.rs[1] : a.rs[0];
    const T *x = reinterpret_cast<const T *>(kv ? a.x[1] : a.x[0]) + row0 * rs + head * D + c * 8;
    float *scales = kv ? a.scale[1] : a.scale[0];
    uint4 v[kPasses];
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
        const int j = p * kRows + r;
        v[p] = j < m ? load8<VEC>(x + j * rs) : make_uint4(0, 0, 0, 0);
    }
    const int page = a.table[(long)s_found[0] * a.max_pages + s_found[1]];
    if (page < 0 || page >= a.n_pages) return;
    const long ps = (long)page * a.kv_heads + head;
    const float old = off ? scales[ps] : 0.f;
    uint32_t top = 0;  // two maxima of magnitudes, as bits
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
        top = __vmaxu2(top, v[p].x & 0x7fff7fffu);
        top = __vmaxu2(top, v[p].y & 0x7fff7fffu);
        top = __vmaxu2(top, v[p].z & 0x7fff7fffu);
        top = __vmaxu2(top, v[p].w & 0x7fff7fffu);
    }
    if (__vcmpgeu2(top, Kv8Bits<T>::inf * 0x10001u)) {
        // infinities saturate and NaN stays NaN, but neither sets the scale
        top = 0;
#pragma unroll
        for (int p = 0; p < kPasses; ++p) {
            const uint32_t w[4] = {v[p].x, v[p].y, v[p].z, v[p].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t b = w[e] & 0x7fff7fffu;
                top = __vmaxu2(top, b & ~__vcmpgeu2(b, Kv8Bits<T>::inf * 0x10001u));
            }
        }
    }
    top = max(top & 0xffffu, top >> 16);
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) s_max[wid] = top;
    __syncthreads();
    top = max(max(s_max[4 * kv], s_max[4 * kv + 1]), max(s_max[4 * kv + 2], s_max[4 * kv + 3]));
    const float scale = fmaxf(old, scale_for(Kv8Bits<T>::value(top)));
    const float inv = 1.0f / scale;  // a power of two: exact
    uint8_t *dst = (kv ? a.pool[1] : a.pool[0]) + (size_t)ps * (kKv8Page * D);
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
        const int j = p * kRows + r;
        if (j < m)
            *reinterpret_cast<uint2 *>(dst + (off + j) * D + c * 8) =
                make_uint2(to_e4m3x2<T>(v[p].x, inv) | to_e4m3x2<T>(v[p].y, inv) << 16,
                           to_e4m3x2<T>(v[p].z, inv) | to_e4m3x2<T>(v[p].w, inv) << 16);
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
    if (t == 0) scales[ps] = scale;
}

// ------------------------------------------------------------------ attention
// Per row and K/V head, G query heads share the keys, 8 NG of them per CTA:
//   S^T[keys x heads] = K Q^T    m16n8k16, keys in M, 8 heads in N
//   P   = exp2(c (S s_k - m) + 11)    m moves only when it is 2^4 behind
//   O^T[dims x heads] += s_v (V^T P)
// The cache is read once (by up to 16 heads per K/V head; more are several CTAs, each of which
// reads it), straight into the registers that hold the A operands:
// the contraction of Q K^T runs over dims in the order in which 16-byte pieces of
// a K row fall to the four lanes of a row group, and V^T is formed from the bytes of four
// keys by permutes, so no shared memory and no barrier stands between HBM and
// the tensor cores.  e4m3 converts to fp16 exactly; bf16 queries are brought to
// fp16 by a power of two per head (their largest value to [2^14, 2^15)).
// P is rounded to fp16 (V's codes convert to it exactly), l sums it before.  The factor 2^11,
// which O and l share, puts P <= 2^15 at the top of fp16's range: a weight down to 2^-25
// of its warp's largest is rounded relative to itself, a smaller one to 2^-36 of it.  (Without
// it the keys behind one that leads them by 18 and has V = 0 counted for nothing.)  O and l
// carry 2^-40 besides, so that no sum passes V's own largest value, which in bf16 is fp32's.
// A warp takes 32 keys at a time and keeps the next 32 keys' K and V in flight.
// The context is shared out in one of these ways:
//   clusters  a cluster of CTAs takes one (row, K/V head) and joins its parts
//             (m, l, O) through distributed shared memory: one launch.  One long row has
//             several; the last of them to arrive joins what they left in the workspace
//   even      the steps of all rows and K/V heads, one after the other, are cut into as
//             many equal runs as CTAs fit on the GPU; a run that ends inside a
//             (row, K/V head) leaves its part in the caller's workspace, and the last of
//             them to arrive joins the parts in their order (a second launch does, where
//             they are many)
constexpr int kAtWarps = 4;
constexpr int kAtKeys = 32;  // keys per warp and step
constexpr float kAtLead = 4.f, kAtBias = 11.f;  // log2 of how far m may fall behind; of what P is multiplied by
constexpr float kAtSum = 0x1p-40f;              // O and l over P V and P

// CTAs that an SM holds, by their registers.
constexpr int kv8_per_sm(int ng, int D) { return ng == 1 ? (D == 64 ? 4 : 3) : (D == 64 ? 3 : 2); }

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
    int heads, kv_heads, G, chunks;  // chunks of 8 NG heads per K/V head
    float scale_log2;
    int vec;       // q rows are 8-byte aligned
    int rows;
    int cluster;   // CTAs that share a (row, K/V head)
    int groups;    // clusters that share it, their parts meeting in the workspace
    int ctas;      // even shares: CTAs of the launch
    int *tickets;  // [kTickets] arrivals of a head group's parts, at the run with its first step (groups: at the
                   // head group); zero between calls.  Null: a second launch joins the parts.
    int *prefix;   // even shares: [rows + 1] cost of the rows before each, per head group (written by CTA 0)
    float *part;   // even shares: [ctas][2][8 NG][D + 4]: O, m, l of a run's part of a head group
                   // groups: [head groups][groups][8 NG][D + 4]
};

// Even shares: a (row, head group) of n steps costs n + kSegCost, the latencies of
// its start and its end (lengths, table, first K and V, queries, the join of the
// warps) being worth kSegCost steps; one without keys costs nothing.  The sum
// `total` of the costs is cut into runs, run c being [c total / runs, (c + 1) total / runs).
// (64 rows of 130 to 8191 keys, 8 K/V heads: 69.2 us with 4, 61.4 with 8, 61.6 with 16.)
constexpr int kSegCost = 8;
constexpr int kTickets = 4096;  // at most so many CTAs
struct Kv8Runs {
    int total, runs, q, r;
    __device__ __forceinline__ Kv8Runs(int total_, int ctas) : total(total_) {
        const int most = (total + kSegCost + 7) / (kSegCost + 8);
        runs = max(1, min(most, ctas));
        q = total / runs;
        r = total % runs;
    }
    // c total / runs, without a 64-bit division (several of those took 0.7 us of a launch)
    __device__ __forceinline__ int begin(int c) const { return c * q + c * r / runs; }
    // the run that has place x of the cost
    __device__ __forceinline__ int owner(int x) const {
        int c = (int)((float)x * (float)runs / (float)total);
        c = max(0, min(c, runs - 1));
        while (c > 0 && begin(c) > x) --c;
        while (c + 1 < runs && begin(c + 1) <= x) ++c;
        return c;
    }
};

__device__ __forceinline__ uint4 ldg_stream16(const void *p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 ldg_stream8(const void *p) {
    uint2 v;
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}
// four e4m3 codes -> two half2, exact
__device__ __forceinline__ void e4m3x4_to_h2x2(uint32_t w, uint32_t &lo, uint32_t &hi) {
    asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
}
__device__ __forceinline__ uint32_t movmatrix_t(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_cluster(const float *p, uint32_t rank) {
    uint32_t a = smem_u32(p), r;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(r) : "memory");
    return v;
}

template <typename T> struct Kv8Q {
    static constexpr bool rescale = false;
};
template <> struct Kv8Q<__nv_bfloat16> {
    static constexpr bool rescale = true;
};

// grid: clusters (cluster * chunks * kv_heads, rows, groups); even shares (ctas)
template <typename T, int D, int NG, bool kEven>
__global__ void __launch_bounds__(kAtWarps * 32, kv8_per_sm(NG, D)) kv8_attn_kernel(const Kv8Attn a) {
    constexpr int HB = 8 * NG;       // heads per CTA
    constexpr int KC = D / 64;       // 16-byte pieces of a K row per lane
    constexpr int MT = D / 16;       // 16-dim tiles of O
    constexpr int VW = D / 32;       // 32-bit words of a V row per lane
    constexpr int kPart = D + 4;     // floats of a part: O, m, l, 2 unused
    __shared__ __align__(16) float s_o[kAtWarps][HB][D];
    __shared__ float s_m[kAtWarps][HB], s_l[kAtWarps][HB];
    __shared__ __align__(16) float s_co[kEven ? 1 : HB][D];
    __shared__ float s_cm[HB], s_cl[HB];  // this CTA's part, read by the cluster
    extern __shared__ int s_prefix[];                              // even shares: [rows + 1]
    __shared__ int s_scan[kAtWarps];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const size_t head_bytes = (size_t)kKv8Page * D, page_bytes = head_bytes * a.kv_heads;
    const int HC = a.kv_heads * a.chunks;
    pdl_wait();
    pdl_trigger();
    auto keys_of = [&](int row) -> long {  // that the row sees
        const int seq = a.seq[row];
        return seq >= 0 && seq < a.n_seqs ? max(0l, min((long)a.pos[row] + 1, (long)a.max_pages * kKv8Page)) : 0;
    };
    int row, rank = 0, hc;
    int u0, u1, step;         // this warp's steps of the segment: u0, u0 + step, ... below u1
    int seg0 = 0;              // even shares: where the run stands in the head group's cost
    int left_cost = 0;         // even shares: what is left of this CTA's run
    Kv8Runs runs(1, 1);
    if (kEven) {
        // cost of the rows before each
        int base = 0;
        for (int r0 = 0; r0 < a.rows; r0 += kAtWarps * 32) {
            const int r = r0 + tid;
            int n = r < a.rows ? (int)((keys_of(r) + kAtKeys - 1) / kAtKeys) : 0;
            if (n) n += kSegCost;
            int in = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, in, o);
                if (lane >= o) in += v;
            }
            __syncthreads();
            if (lane == 31) s_scan[warp] = in;
            __syncthreads();
            int before = base + in - n;
#pragma unroll
            for (int w = 0; w < kAtWarps; ++w) {
                if (w < warp) before += s_scan[w];
                base += s_scan[w];
            }
            if (r < a.rows) s_prefix[r] = before;
        }
        if (tid == 0) s_prefix[a.rows] = base;
        __syncthreads();
        if (blockIdx.x == 0 && !a.tickets)
            for (int r = tid; r <= a.rows; r += kAtWarps * 32) a.prefix[r] = s_prefix[r];
        // rows that see nothing
        for (int r = blockIdx.x; r < a.rows; r += a.ctas)
            if (s_prefix[r] == s_prefix[r + 1])
                for (int x = tid; x < a.heads * D; x += kAtWarps * 32)
                    reinterpret_cast<T *>(a.out)[(long)r * a.out_rs + x] = from_float<T>(0.f);
        runs = Kv8Runs(base * HC, a.ctas);
        if (base == 0 || blockIdx.x >= runs.runs) return;
        const int b0 = runs.begin(blockIdx.x);
        left_cost = runs.begin(blockIdx.x + 1) - b0;
        int lo = 0, hi = a.rows;  // the last row that starts at or before b0
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s_prefix[mid] * HC <= b0)
                lo = mid;
            else
                hi = mid;
        }
        row = lo;
        const int n = s_prefix[row + 1] - s_prefix[row];
        const int rem = b0 - s_prefix[row] * HC;
        hc = rem / n;
        seg0 = rem % n;
    } else {
        rank = blockIdx.x % a.cluster;
        hc = blockIdx.x / a.cluster;
        row = blockIdx.y;
    }
    for (;;) {  // segments of this CTA: parts of one (row, K/V head, chunk of heads) each
    const int kvh = hc / a.chunks, h0 = (hc % a.chunks) * HB;  // first head, within the group
    const long len = keys_of(row);
    const int *table = a.table + (long)(len > 0 ? a.seq[row] : 0) * a.max_pages;
    const int units = (int)((len + kAtKeys - 1) / kAtKeys);
    const int cut = min(units + kSegCost, seg0 + left_cost);  // even shares: where the run leaves it
    const int first = max(seg0 - kSegCost, 0);
    if (kEven) {
        u0 = first + warp;
        u1 = cut - kSegCost;
        step = kAtWarps;
    } else {
        u0 = (blockIdx.z * a.cluster + rank) * kAtWarps + warp;
        u1 = units;
        step = a.groups * a.cluster * kAtWarps;
    }

    uint4 kr[4][KC];   // K: rows g, g + 8, g + 16, g + 24 of the step's keys
    uint32_t vr[8][VW];  // V: keys 2t, 2t + 1, 2t + 8, 2t + 9 of both 16-key tiles; dims VW * 4 * g ..
    int page = -1, next_page = -1;  // of the step in registers, of the one after
    float ks = 0.f, vs = 0.f;
    auto page_of = [&](int u) -> int {
        if (u >= u1) return -1;
        const int p = table[u >> 1];
        return p >= 0 && p < a.n_pages ? p : -1;
    };
    auto load_k = [&](int u, int p) {
        if (p < 0) return;
        const uint8_t *b = a.kpool + p * page_bytes + kvh * head_bytes + (u & 1) * (kAtKeys * D) + g * D + t * 16;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < KC; ++c) kr[r][c] = ldg_stream16(b + r * 8 * D + c * 64);
    };
    auto load_v = [&](int u, int p) {
        if (p < 0) return;
        const uint8_t *b = a.vpool + p * page_bytes + kvh * head_bytes + (u & 1) * (kAtKeys * D) + 2 * t * D + g * (VW * 4);
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const uint8_t *x = b + ((r >> 2) * 16 + (r & 1) + ((r >> 1) & 1) * 8) * D;
            if (VW == 4) {
                const uint4 v = ldg_stream16(x);
                vr[r][0] = v.x, vr[r][1] = v.y, vr[r][VW > 2 ? 2 : 0] = v.z, vr[r][VW > 2 ? 3 : 0] = v.w;
            } else {
                const uint2 v = ldg_stream8(x);
                vr[r][0] = v.x, vr[r][1] = v.y;
            }
        }
    };
    page = page_of(u0);
    next_page = page_of(u0 + step);
    load_k(u0, page);
    load_v(u0, page);
    if (page >= 0) {
        ks = a.kscale[(long)page * a.kv_heads + kvh];
        vs = a.vscale[(long)page * a.kv_heads + kvh];
    }

    // ---- queries: B operand, lane (g, t) holds head g, dims 64 c + 16 t + 4 k .. + 3
    uint32_t qb[NG][KC * 4][2];
    float c0[NG], c1[NG];  // of heads 2t, 2t + 1: what a product of codes counts, in log2
#pragma unroll
    for (int n = 0; n < NG; ++n) {
        const int h = h0 + n * 8 + g;
        const T *q = reinterpret_cast<const T *>(a.q) + (long)row * a.q_rs + (long)(kvh * a.G + h) * D + 16 * t;
        T x[KC * 4][4];
#pragma unroll
        for (int k = 0; k < KC * 4; ++k) {
            const T *src = q + (k >> 2) * 64 + (k & 3) * 4;
            uint2 u = make_uint2(0, 0);
            if (h < a.G) {
                if (a.vec) {
                    u = *reinterpret_cast<const uint2 *>(src);
                } else {
                    const unsigned short *e = reinterpret_cast<const unsigned short *>(src);
                    u.x = e[0] | (uint32_t)e[1] << 16;
                    u.y = e[2] | (uint32_t)e[3] << 16;
                }
            }
            *reinterpret_cast<uint2 *>(x[k]) = u;
        }
        float f = 1.f;
        if (Kv8Q<T>::rescale) {
            float m = 0.f;
#pragma unroll
            for (int k = 0; k < KC * 4; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) m = fmaxf(m, fabsf(to_float(x[k][e])));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
            const int e = max((int)(__float_as_uint(m) >> 23) - 127, -100);
            f = __uint_as_float((uint32_t)(14 - e + 127) << 23);
#pragma unroll
            for (int k = 0; k < KC * 4; ++k)
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const __half2 v = __floats2half2_rn(to_float(x[k][2 * p]) * f, to_float(x[k][2 * p + 1]) * f);
                    qb[n][k][p] = *reinterpret_cast<const uint32_t *>(&v);
                }
            f = __uint_as_float((uint32_t)(e - 14 + 127) << 23);
        } else {
#pragma unroll
            for (int k = 0; k < KC * 4; ++k)
#pragma unroll
                for (int p = 0; p < 2; ++p) qb[n][k][p] = reinterpret_cast<const uint32_t *>(x[k])[p];
        }
        c0[n] = __shfl_sync(0xffffffffu, f, 8 * t) * a.scale_log2;
        c1[n] = __shfl_sync(0xffffffffu, f, 8 * t + 4) * a.scale_log2;
    }

    float o[NG][MT][4], m0[NG], m1[NG], l0[NG], l1[NG];
#pragma unroll
    for (int n = 0; n < NG; ++n) {
        m0[n] = m1[n] = -INFINITY;
        l0[n] = l1[n] = 0.f;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][i][e] = 0.f;
    }
    for (int u = u0; u < u1; u += step) {
        const int cur = page;
        const float cks = ks, cvs = vs * kAtSum;
        page = next_page;
        next_page = page_of(u + 2 * step);
        if (page >= 0) {
            ks = a.kscale[(long)page * a.kv_heads + kvh];
            vs = a.vscale[(long)page * a.kv_heads + kvh];
        }
        uint32_t pb[NG][2][2];
        if (cur >= 0) {
            // ---- scores of 32 keys
            float s[NG][2][4];
#pragma unroll
            for (int n = 0; n < NG; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[n][i][e] = 0.f;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int k = 0; k < KC * 4; ++k) {
                    const uint32_t w0 = reinterpret_cast<const uint32_t *>(&kr[2 * i][k >> 2])[k & 3];
                    const uint32_t w1 = reinterpret_cast<const uint32_t *>(&kr[2 * i + 1][k >> 2])[k & 3];
                    uint32_t a0, a1, a2, a3;
                    e4m3x4_to_h2x2(w0, a0, a2);
                    e4m3x4_to_h2x2(w1, a1, a3);
#pragma unroll
                    for (int n = 0; n < NG; ++n) mma_f16(s[n][i], a0, a1, a2, a3, qb[n][k][0], qb[n][k][1]);
                }
            load_k(u + step, page);
            // ---- softmax: lane holds heads 2t (e = 0, 2) and 2t + 1 (1, 3), keys g (e < 2) and g + 8
            const int left = (int)min(len - (long)u * kAtKeys, (long)kAtKeys);  // keys that the row sees
            bool move = false;
#pragma unroll
            for (int n = 0; n < NG; ++n) {
                const float f0 = c0[n] * cks, f1 = c1[n] * cks;
                float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bool seen = i * 16 + (e >> 1) * 8 + g < left;
                        s[n][i][e] = seen ? s[n][i][e] * ((e & 1) ? f1 : f0) : -INFINITY;
                        if (e & 1)
                            x1 = fmaxf(x1, s[n][i][e]);
                        else
                            x0 = fmaxf(x0, s[n][i][e]);
                    }
                move |= x0 - m0[n] > kAtLead || x1 - m1[n] > kAtLead;
                if (__any_sync(0xffffffffu, move)) {
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) {
                        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, d));
                        x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, d));
                    }
                    const float y0 = fmaxf(m0[n], x0), y1 = fmaxf(m1[n], x1);
                    const float r0 = m0[n] == y0 || m0[n] == -INFINITY ? 1.f : ex2(m0[n] - y0);
                    const float r1 = m1[n] == y1 || m1[n] == -INFINITY ? 1.f : ex2(m1[n] - y1);
                    m0[n] = y0;
                    m1[n] = y1;
                    l0[n] *= r0;
                    l1[n] *= r1;
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        o[n][i][0] *= r0;
                        o[n][i][1] *= r1;
                        o[n][i][2] *= r0;
                        o[n][i][3] *= r1;
                    }
                }
                // (rounded up, so that P <= 2^15 holds for scores of any size)
                const float b0 = m0[n] == -INFINITY ? 0.f : __fsub_ru(m0[n], kAtBias);
                const float b1 = m1[n] == -INFINITY ? 0.f : __fsub_ru(m1[n], kAtBias);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[n][i][e] = ex2(s[n][i][e] - ((e & 1) ? b1 : b0));
                        if (e & 1)
                            l1[n] += s[n][i][e];
                        else
                            l0[n] += s[n][i][e];
                    }
                    // P^T as the B operand: (key, heads) pairs -> (head, keys) pairs
                    const __half2 lo = __floats2half2_rn(s[n][i][0], s[n][i][1]);
                    const __half2 hi = __floats2half2_rn(s[n][i][2], s[n][i][3]);
                    pb[n][i][0] = movmatrix_t(*reinterpret_cast<const uint32_t *>(&lo));
                    pb[n][i][1] = movmatrix_t(*reinterpret_cast<const uint32_t *>(&hi));
                }
            }
            if (left < kAtKeys) {  // codes behind the end may be anything, NaN included
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if ((r >> 2) * 16 + 2 * t + (r & 1) + ((r >> 1) & 1) * 8 >= left)
#pragma unroll
                        for (int w = 0; w < VW; ++w) vr[r][w] = 0;
            }
            // ---- O^T += s_v V^T P: dims VW 4 g + 4 w + 2 j (row g) and + 1 (row g + 8) in tile 2 w + j
#pragma unroll
            for (int w = 0; w < VW; ++w) {
                float acc[NG][2][4];
#pragma unroll
                for (int n = 0; n < NG; ++n)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[n][j][e] = 0.f;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t x[2][2];  // [keys 2t, 2t + 1 | 2t + 8, 2t + 9][dims 0, 1 | 2, 3], key pairs per dim
#pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        x[p][0] = __byte_perm(vr[4 * i + 2 * p][w], vr[4 * i + 2 * p + 1][w], 0x5140);
                        x[p][1] = __byte_perm(vr[4 * i + 2 * p][w], vr[4 * i + 2 * p + 1][w], 0x7362);
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        uint32_t a0, a1, a2, a3;
                        e4m3x4_to_h2x2(x[0][j], a0, a1);
                        e4m3x4_to_h2x2(x[1][j], a2, a3);
#pragma unroll
                        for (int n = 0; n < NG; ++n) mma_f16(acc[n][j], a0, a1, a2, a3, pb[n][i][0], pb[n][i][1]);
                    }
                }
#pragma unroll
                for (int n = 0; n < NG; ++n)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[n][2 * w + j][e] = fmaf(acc[n][j][e], cvs, o[n][2 * w + j][e]);
            }
        } else {
            load_k(u + step, page);
        }
        load_v(u + step, page);
    }

    // ---- join the warps, then the cluster's CTAs or (another launch) the runs
#pragma unroll
    for (int n = 0; n < NG; ++n) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
            l0[n] += __shfl_xor_sync(0xffffffffu, l0[n], d);
            l1[n] += __shfl_xor_sync(0xffffffffu, l1[n], d);
        }
        l0[n] *= kAtSum;
        l1[n] *= kAtSum;
        const int h = n * 8 + 2 * t;
        if (g == 0) {
            s_m[warp][h] = m0[n];
            s_m[warp][h + 1] = m1[n];
            s_l[warp][h] = l0[n];
            s_l[warp][h + 1] = l1[n];
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int d = VW * 4 * g + 2 * i;
            *reinterpret_cast<float2 *>(&s_o[warp][h][d]) = make_float2(o[n][i][0], o[n][i][2]);
            *reinterpret_cast<float2 *>(&s_o[warp][h + 1][d]) = make_float2(o[n][i][1], o[n][i][3]);
        }
    }
    __syncthreads();
    const int nh = kEven && u1 <= first ? 0 : min(HB, a.G - h0);  // 0: the run ends before the first step
    const bool whole = !kEven || (first == 0 && u1 == units);
    float *part = kEven ? a.part + ((long)blockIdx.x * 2 + (first == 0)) * HB * kPart : nullptr;
    // the warps' parts relative to the largest maximum
    __shared__ float s_f[kAtWarps][HB];
    if (tid < HB) {
        float m = s_m[0][tid], l = 0.f;
#pragma unroll
        for (int w = 1; w < kAtWarps; ++w) m = fmaxf(m, s_m[w][tid]);
#pragma unroll
        for (int w = 0; w < kAtWarps; ++w) {
            const float mw = s_m[w][tid], lw = s_l[w][tid];
            const float f = mw == -INFINITY ? (lw != lw ? 1.f : 0.f) : ex2(mw - m);
            s_f[w][tid] = f;
            l += lw * f;
        }
        s_cm[tid] = m;
        s_cl[tid] = l;
    }
    __syncthreads();
    for (int x = tid; x < nh * (D / 4); x += kAtWarps * 32) {
        const int h = x / (D / 4), d = x % (D / 4) * 4;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kAtWarps; ++w) {
            const float f = s_f[w][h];
            const float4 o4 = *reinterpret_cast<const float4 *>(&s_o[w][h][d]);
            v.x += o4.x * f, v.y += o4.y * f, v.z += o4.z * f, v.w += o4.w * f;
        }
        if (!kEven && a.cluster > 1) {
            *reinterpret_cast<float4 *>(&s_co[kEven ? 0 : h][d]) = v;
        } else if (whole) {
            const float l = s_cl[h], inv = l > 0.f || l != l ? 1.f / l : 0.f;
            T *dst = reinterpret_cast<T *>(a.out) + (long)row * a.out_rs + (long)(kvh * a.G + h0 + h) * D + d;
            dst[0] = from_float<T>(v.x * inv);
            dst[1] = from_float<T>(v.y * inv);
            dst[2] = from_float<T>(v.z * inv);
            dst[3] = from_float<T>(v.w * inv);
        } else {
            float *p = part + h * kPart;
            *reinterpret_cast<float4 *>(p + d) = v;
            if (d == 0) *reinterpret_cast<float2 *>(p + D) = make_float2(s_cm[h], s_cl[h]);
        }
    }
    if (!kEven && a.cluster > 1) {
        cluster_sync_all();
        const int share = (nh * D + a.cluster - 1) / a.cluster;
        const int x1 = min(nh * D, (rank + 1) * share);
        T *out = reinterpret_cast<T *>(a.out) + (long)row * a.out_rs + (long)(kvh * a.G + h0) * D;
        float *group0 = a.part + (long)hc * a.groups * HB * kPart;
        for (int x = rank * share + tid; x < x1; x += kAtWarps * 32) {
            const int h = x / D, d = x % D;
            float m = -INFINITY;
            for (int c = 0; c < a.cluster; ++c) m = fmaxf(m, ld_cluster(&s_cm[h], c));
            float l = 0.f, v = 0.f;
            for (int c = 0; c < a.cluster; ++c) {
                const float mc = ld_cluster(&s_cm[h], c), lc = ld_cluster(&s_cl[h], c);
                const float f = mc == -INFINITY ? (lc != lc ? 1.f : 0.f) : ex2(mc - m);
                l += lc * f;
                v += ld_cluster(&s_co[kEven ? 0 : h][d], c) * f;
            }
            if (a.groups > 1) {
                float *p = group0 + ((long)blockIdx.z * HB + h) * kPart;
                p[d] = v;
                if (d == 0) *reinterpret_cast<float2 *>(p + D) = make_float2(m, l);
            } else {
                out[h * D + d] = from_float<T>(l > 0.f || l != l ? v / l : 0.f);
            }
        }
        if (a.groups > 1) {
            // the last cluster to arrive joins the parts, in their order
            __threadfence();
            cluster_sync_all();
            __shared__ float s_last;
            if (rank == 0 && tid == 0) {
                const bool last = atomicAdd(&a.tickets[hc], 1) == a.groups - 1;
                if (last) a.tickets[hc] = 0;
                s_last = last ? 1.f : 0.f;
            }
            cluster_sync_all();
            if (ld_cluster(&s_last, 0) != 0.f) {
                __threadfence();
                float2(*s_ml)[HB] = reinterpret_cast<float2(*)[HB]>(&s_o[0][0][0]);  // [groups][head]
                for (int x = tid; x < a.groups * HB; x += kAtWarps * 32) {
                    const int c = x / HB, h = x % HB;
                    if (h < nh)
                        s_ml[c][h] = __ldcg(reinterpret_cast<const float2 *>(group0 + ((long)c * HB + h) * kPart + D));
                }
                __syncthreads();
                for (int x = rank * share + tid; x < x1; x += kAtWarps * 32) {
                    const int h = x / D, d = x % D;
                    const float *p = group0 + h * kPart + d;
                    float m = -INFINITY, l = 0.f, v = 0.f;
                    for (int c = 0; c < a.groups; ++c) m = fmaxf(m, s_ml[c][h].x);
#pragma unroll 16
                    for (int c = 0; c < a.groups; ++c) {
                        const float o = __ldcg(p + c * (HB * kPart));
                        const float2 ml = s_ml[c][h];
                        const float f = ml.x == -INFINITY ? (ml.y != ml.y ? 1.f : 0.f) : ex2(ml.x - m);
                        l += ml.y * f;
                        v += o * f;
                    }
                    out[h * D + d] = from_float<T>(l > 0.f || l != l ? v / l : 0.f);
                }
            }
        }
        cluster_sync_all();  // no CTA leaves while its part is read
    }
    if (!kEven) return;
    if (nh > 0 && !whole && a.tickets) {
        __shared__ int s_last;
        const int n = units + kSegCost;
        const int s0 = s_prefix[row] * HC + hc * n;
        const int c0 = runs.owner(s0 + kSegCost), c1 = runs.owner(s0 + n - 1);
        __threadfence();
        __syncthreads();
        if (tid == 0) {
            s_last = atomicAdd(&a.tickets[c0], 1) == c1 - c0;
            if (s_last) a.tickets[c0] = 0;
        }
        __syncthreads();
        if (s_last) {
            __threadfence();
            // part 0 begins the head group in run c0, the others continue it
            auto at = [&](int c) { return a.part + ((long)(c0 + c) * 2 + (c == 0)) * HB * kPart; };
            const int parts = c1 - c0 + 1;
            constexpr int NV = HB * D / 4 / (kAtWarps * 32);  // float4 outputs per thread
            float4 v[NV];
            float m[NV], l[NV];
#pragma unroll
            for (int y = 0; y < NV; ++y) {
                v[y] = make_float4(0.f, 0.f, 0.f, 0.f);
                m[y] = -INFINITY;
                l[y] = 0.f;
            }
            float(*s_pm)[2][HB] = reinterpret_cast<float(*)[2][HB]>(&s_o[0][0][0]);  // [32 parts][m, l][head]
            for (int cb = 0; cb < parts; cb += 32) {
                const int nc = min(32, parts - cb);
                __syncthreads();
                for (int x = tid; x < nc * 2 * HB; x += kAtWarps * 32) {
                    const int c = x / (2 * HB), k = x / HB & 1, h = x % HB;
                    s_pm[c][k][h] = h < nh ? __ldcg(at(cb + c) + h * kPart + D + k) : 0.f;
                }
                __syncthreads();
#pragma unroll
                for (int y = 0; y < NV; ++y) {
                    const int x = tid + y * kAtWarps * 32, h = x / (D / 4), d = x % (D / 4) * 4;
                    float mn = m[y];
                    for (int c = 0; c < nc; ++c) mn = fmaxf(mn, s_pm[c][0][h]);
                    const float f = m[y] == -INFINITY ? 1.f : ex2(m[y] - mn);  // with m = -inf, v and l are 0
                    m[y] = mn;
                    l[y] *= f;
                    v[y].x *= f, v[y].y *= f, v[y].z *= f, v[y].w *= f;
#pragma unroll 4
                    for (int c = 0; c < nc; ++c) {
                        const float4 o = __ldcg(reinterpret_cast<const float4 *>(at(cb + c) + h * kPart + d));
                        const float mc = s_pm[c][0][h], lc = s_pm[c][1][h];
                        const float fc = mc == -INFINITY ? (lc != lc ? 1.f : 0.f) : ex2(mc - mn);
                        l[y] += lc * fc;
                        v[y].x += o.x * fc, v[y].y += o.y * fc, v[y].z += o.z * fc, v[y].w += o.w * fc;
                    }
                }
            }
#pragma unroll
            for (int y = 0; y < NV; ++y) {
                const int x = tid + y * kAtWarps * 32, h = x / (D / 4), d = x % (D / 4) * 4;
                if (h >= nh) continue;
                const float inv = l[y] > 0.f || l[y] != l[y] ? 1.f / l[y] : 0.f;
                T *o = reinterpret_cast<T *>(a.out) + (long)row * a.out_rs + (long)(kvh * a.G + h0 + h) * D + d;
                o[0] = from_float<T>(v[y].x * inv);
                o[1] = from_float<T>(v[y].y * inv);
                o[2] = from_float<T>(v[y].z * inv);
                o[3] = from_float<T>(v[y].w * inv);
            }
        }
    }
    left_cost -= cut - seg0;
    if (left_cost <= 0) return;
    seg0 = 0;
    if (++hc == HC) {
        hc = 0;
        do ++row;
        while (s_prefix[row] == s_prefix[row + 1]);
    }
    __syncthreads();  // the parts in shared memory have been read
    }
}

// Even shares: out = sum of O 2^(m - max) over the runs that share a (row, head), over the
// sum of l 2^(m - max).  grid (heads, rows, dim blocks), 256 threads.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv8_join_kernel(T *__restrict__ out, long out_rs, const float *__restrict__ part,
                                                       const int *__restrict__ prefix, int rows, int ctas, int G,
                                                       int chunks, int kv_heads, int HB) {
    extern __shared__ float s_w[];  // [2][ctas]: m, then 2^(m - max), and l of each part
    __shared__ float s_v[256], s_r[8];
    const int h = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, dims = D / gridDim.z, groups = 256 / dims;
    const int d = blockIdx.z * dims + tid % dims, q = tid / dims;
    const int HC = kv_heads * chunks, hl = h % G, hc = h / G * chunks + hl / HB;
    pdl_wait();
    pdl_trigger();
    const int p0 = prefix[row], n = prefix[row + 1] - p0;
    const int total = prefix[rows] * HC;
    if (n == 0) return;
    const Kv8Runs cut(total, ctas);
    const int s0 = p0 * HC + hc * n;
    // the runs with its first and its last step
    const int c0 = cut.owner(s0 + kSegCost), c1 = cut.owner(s0 + n - 1);
    if (c0 == c1) return;  // one run had all of it
    // the first run's part begins with the head group, the others continue it
    const float *base = part + ((long)c0 * 2 * HB + hl % HB) * (D + 4);
    const long next = 2l * HB * (D + 4), begins = (long)HB * (D + 4);
    auto block = [&](float v, bool sum) -> float {  // over the 256 threads
        v = sum ? warp_sum(v) : warp_max(v);
        __syncthreads();
        if ((tid & 31) == 0) s_r[tid >> 5] = v;
        __syncthreads();
        v = s_r[0];
#pragma unroll
        for (int w = 1; w < 8; ++w) v = sum ? v + s_r[w] : fmaxf(v, s_r[w]);
        return v;
    };
    float m = -INFINITY;
    for (int c = tid; c <= c1 - c0; c += 256) {
        const float *p = base + c * next + (c == 0 ? begins : 0) + D;
        s_w[c] = p[0];
        s_w[ctas + c] = p[1];
        m = fmaxf(m, s_w[c]);
    }
    m = block(m, false);
    float l = 0.f;
    for (int c = tid; c <= c1 - c0; c += 256) {
        const float mc = s_w[c], lc = s_w[ctas + c];
        const float f = mc == -INFINITY ? (lc != lc ? 1.f : 0.f) : ex2(mc - m);
        s_w[c] = f;
        l += lc * f;
    }
    l = block(l, true);
    float v = 0.f;
    if (q == 0) v = base[begins + d] * s_w[0];
#pragma unroll 8
    for (int c = 1 + q; c <= c1 - c0; c += groups) v += base[c * next + d] * s_w[c];
    s_v[tid] = v;
    __syncthreads();
    if (q == 0) {
        for (int k = 1; k < groups; ++k) v += s_v[k * dims + tid];
        out[row * out_rs + (long)h * D + d] = from_float<T>(l > 0.f || l != l ? v / l : 0.f);
    }
}

// How a call's context is shared out.
constexpr int kEvenMaxRows = 2048;  // their prefix sums lie in shared memory
constexpr int kMaxGroups = 64;      // their maxima and sums lie in shared memory
struct Kv8Split {
    int ng, chunks, cluster;
    int groups;  // clusters to a head group
    int ctas;    // even shares (0: clusters)
    bool wide;   // even shares: more than 16 parts to a head group, which a second launch joins
};
Kv8Split kv8_split(int rows, int max_len, int max_pages, int heads, int kv_heads, int D, int sms, bool workspace) {
    Kv8Split s;
    const int G = heads / kv_heads;
    s.ng = G <= 8 ? 1 : 2;
    s.chunks = (G + 8 * s.ng - 1) / (8 * s.ng);
    const long pairs = (long)rows * kv_heads * s.chunks;
    const int units = max_len > 0 ? (max_len - 1) / kAtKeys + 1 : 1;
    const long ctas = (long)kv8_per_sm(s.ng, D) * sms;
    // Clusters: as many CTAs each as fill the machine in one wave and have a step for every
    // warp.  Equal runs where that leaves a warp more than 12 steps in a row, or rows to wait
    // for one another in waves (a wave's steps are then many, too).  us, clusters / runs:
    //   16 rows of 4096, 8 K/V heads (11 steps)   28.9 / 32.0     8 of 2048   13.2 / 17.6
    //   64 rows of 130 to 8191, 8 heads           81.2 / 53.5     64 of 1024  34.2 / 34.2
    const int useful = (units + kAtWarps - 1) / kAtWarps;
    const long one_wave = ctas / pairs > 0 ? ctas / pairs : 1;
    const long most = useful < 8 ? useful : 8;
    auto clamp = [&](long c) -> int { return (int)(c < most ? c : most); };
    s.cluster = clamp(one_wave);
    // a pair's parts are joined by the last run to arrive, up to 16 of them on average
    s.wide = pairs * 16 < ctas;
    // (costs are added up in 32 bits)
    s.ctas = workspace && rows <= kEvenMaxRows && units > 12l * kAtWarps * s.cluster &&
                     pairs * (2l * max_pages + kSegCost) < (1l << 30) && ctas <= kTickets
                 ? (int)ctas : 0;
    // One row that leaves a cluster's warps more than 4 steps (8 of head_dim 64: with 6, 9.8 us in one
    // cluster, 10.4 in several): several clusters of 8 to a head
    // group, until a warp has 1 step (head_dim 64) or 2 (128: 8192 keys, 32 / 8 heads take
    // 14.5 us with 2, 15.2 with 1; 16384 keys, 16 / 4 heads of 64 12.6 and 10.5), or no more fit
    // at once (7 of 8 CTAs, for a cluster takes its SMs from one part of the GPU).
    // us, one cluster or equal runs / several clusters:
    //   8192 keys, 8 / 1 heads of 128   13.9 / 11.3     32768   15.4 / 12.5    131071   21.2 / 19.0
    //   8192 keys, 32 / 8 heads of 128  15.8 / 14.5     16384   20.0 / 17.5     65536   34.2 / 32.9
    s.groups = 1;
    const long fit = ctas * 7 / 64 / pairs;
    if (workspace && rows == 1 && fit > 1 && units > (D == 64 ? 8 : 4) * kAtWarps * s.cluster) {
        const int each = 8 * kAtWarps * (D == 64 ? 1 : 2), want = (units + each - 1) / each;
        s.cluster = 8;
        s.groups = (int)(fit < kMaxGroups ? fit : kMaxGroups);
        if (want < s.groups) s.groups = want;
        s.ctas = 0;
        s.wide = false;
        return s;
    }
    // clusters all the same: at most 16 steps per warp, as far as 8 CTAs go
    if (!s.ctas && clamp(units / (16 * kAtWarps) + 1) > s.cluster) s.cluster = clamp(units / (16 * kAtWarps) + 1);
    return s;
}
long long kv8_ws_bytes(const Kv8Split &s, int rows, int head_groups, int D) {
    const long long prefix = (4ll * (rows + 1) + 15) / 16 * 16;
    const long long parts = s.ctas ? 2ll * s.ctas : s.groups > 1 ? (long long)s.groups * head_groups : 0;
    return parts ? 4ll * kTickets + prefix + 4ll * parts * 8 * s.ng * (D + 4) : 0;
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

template <typename T, int D, int NG> cudaError_t launch_attn_ng(const Kv8Attn &a, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kAtWarps * 32);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = g_rt.pdl ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    if (a.ctas == 0) {
        cfg.gridDim = dim3(a.cluster * a.chunks * a.kv_heads, a.rows, a.groups);
        cfg.numAttrs = 2;
        return cudaLaunchKernelEx(&cfg, kv8_attn_kernel<T, D, NG, false>, a);
    }
    cfg.gridDim = dim3(a.ctas);
    cfg.dynamicSmemBytes = 4 * (size_t)(a.rows + 1);
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kv8_attn_kernel<T, D, NG, true>, a);
    if (e != cudaSuccess || a.tickets) return e;
    cfg.gridDim = dim3(a.heads, a.rows, (long)a.heads * a.rows >= g_rt.num_sms / 2 ? 4 : 8);
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = 8 * (size_t)a.ctas;
    return cudaLaunchKernelEx(&cfg, kv8_join_kernel<T, D>, (T *)a.out, a.out_rs, (const float *)a.part,
                              (const int *)a.prefix, a.rows, a.ctas, a.G, a.chunks, a.kv_heads, 8 * NG);
}

template <typename T, int D> cudaError_t launch_attn(const Kv8Attn &a, int ng, cudaStream_t s) {
    return ng == 1 ? launch_attn_ng<T, D, 1>(a, s) : launch_attn_ng<T, D, 2>(a, s);
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
    if ((((uintptr_t)k | (uintptr_t)v) % 2) ||
        (((uintptr_t)kscale | (uintptr_t)vscale | (uintptr_t)starts | (uintptr_t)ctx | (uintptr_t)block_table) % 4))
        return fail("wk_kv8_store: misaligned argument");
    if (g_rt.device < 0) return fail("wk_kv8_store: cuda_init() has not been called");
    DeviceGuard guard;
    Kv8Store a{{(uint8_t *)kpool, (uint8_t *)vpool}, {kscale, vscale}, n_pages, {k, v}, {k_rs, v_rs}, starts, ctx, n,
               rows, block_table, max_pages, kv_heads};
    // base(n) of the kernel, with all rows
    const long long most = (long long)rows / kKv8Page + 2ll * n;
    const int units = (int)(most < rows ? most : rows);
    cudaStream_t s = stream();
    cudaError_t e;
    if (dtype == kF16)
        e = head_dim == 64 ? launch_store<__half, 64>(a, units, s) : launch_store<__half, 128>(a, units, s);
    else
        e = head_dim == 64 ? launch_store<__nv_bfloat16, 64>(a, units, s) : launch_store<__nv_bfloat16, 128>(a, units, s);
    if (e != cudaSuccess) return fail_cuda("wk_kv8_store", e);
    return 0;
}

long long wk_kv8_attention_ws(int rows, int max_len, int n_heads, int kv_heads, int head_dim) {
    if (rows < 1 || max_len < 1 || kv_heads < 1 || n_heads < 1 || n_heads % kv_heads || head_dim < 1) return 0;
    const int sms = g_rt.num_sms > 0 ? g_rt.num_sms : 148;
    const Kv8Split sp = kv8_split(rows, max_len, 1, n_heads, kv_heads, head_dim, sms, true);
    return kv8_ws_bytes(sp, rows, kv_heads * sp.chunks, head_dim);
}

int wk_kv8_attention(void *out, long out_rs, const void *q, long q_rs, const void *kpool, const void *vpool,
                     const float *kscale, const float *vscale, int n_pages, const int *block_table, int n_seqs,
                     int max_pages, const int *seq, const int *pos, int rows, int max_len, int n_heads, int kv_heads,
                     int head_dim, int dtype, void *ws, long long ws_bytes) {
    if (rows < 0 || rows > 65535 || n_pages < 1 || n_seqs < 1 || max_pages < 1 || max_pages > 1 << 25 ||
        max_len < 0 || ws_bytes < 0)
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
    if ((uintptr_t)ws % 16) return fail("wk_kv8_attention: workspace must be 16-byte aligned");
    if ((((uintptr_t)out | (uintptr_t)q) % 2) ||
        (((uintptr_t)kscale | (uintptr_t)vscale | (uintptr_t)block_table | (uintptr_t)seq | (uintptr_t)pos) % 4))
        return fail("wk_kv8_attention: misaligned argument");
    if (g_rt.device < 0) return fail("wk_kv8_attention: cuda_init() has not been called");
    DeviceGuard guard;
    Kv8Split sp = kv8_split(rows, max_len, max_pages, n_heads, kv_heads, head_dim, g_rt.num_sms, ws != nullptr);
    if (ws_bytes < kv8_ws_bytes(sp, rows, kv_heads * sp.chunks, head_dim))
        sp = kv8_split(rows, max_len, max_pages, n_heads, kv_heads, head_dim, g_rt.num_sms, false);
    Kv8Attn a;
    a.out = out;
    a.out_rs = out_rs;
    a.q = q;
    a.q_rs = q_rs;
    a.kpool = (const uint8_t *)kpool;
    a.vpool = (const uint8_t *)vpool;
    a.kscale = kscale;
    a.vscale = vscale;
    a.n_pages = n_pages;
    a.table = block_table;
    a.n_seqs = n_seqs;
    a.max_pages = max_pages;
    a.seq = seq;
    a.pos = pos;
    a.heads = n_heads;
    a.kv_heads = kv_heads;
    a.G = n_heads / kv_heads;
    a.chunks = sp.chunks;
    a.scale_log2 = 1.4426950408889634f / sqrtf((float)head_dim);
    a.vec = ((uintptr_t)q % 8) == 0 && q_rs % 4 == 0;
    a.cluster = sp.cluster;
    a.groups = sp.groups;
    a.rows = rows;
    a.ctas = sp.ctas;
    a.tickets = sp.wide ? nullptr : (int *)ws;
    a.prefix = (int *)ws + kTickets;
    a.part = (float *)((char *)ws + 4ll * kTickets + (4ll * (rows + 1) + 15) / 16 * 16);
    cudaStream_t s = stream();
    cudaError_t e;
    if (dtype == kF16)
        e = head_dim == 64 ? launch_attn<__half, 64>(a, sp.ng, s) : launch_attn<__half, 128>(a, sp.ng, s);
    else
        e = head_dim == 64 ? launch_attn<__nv_bfloat16, 64>(a, sp.ng, s)
                           : launch_attn<__nv_bfloat16, 128>(a, sp.ng, s);
    if (e != cudaSuccess) return fail_cuda("wk_kv8_attention", e);
    return 0;
}

}  // extern "C"
