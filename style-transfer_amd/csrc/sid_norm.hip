// Group normalisation with an activation over channels-last tensors, forward and backward.
//
//   x (B, N, C) with C contiguous (an NCHW tensor in channels-last memory: N = H*W), G groups of Cg = C/G channels
//   mean, rstd per (image, group) over N*Cg values;  xh = (x - mean) rstd;  z = xh w + b;  y = act(z)
//   dz = dy act'(z);  db = sum dz;  dw = sum dz xh            (over images and rows, per channel)
//   dx = rstd (dz w - s1 - xh s2),   s1 = mean over the group of dz w,  s2 = mean over the group of dz w xh
//
// Both directions are bound by memory: forward reads x and writes y, backward reads x and dy and writes dx.
// Two forms, chosen by make_plan():
//   resident  one workgroup per (image, group) keeps its slice (N rows of Cg channels) in registers between the
//             statistics and the output: everything is read once, in one launch, and the variance is taken of
//             centred values.  A row's slice is short (20 bytes at Cg = 10, bf16), so neighbouring groups share
//             cache lines: workgroups that follow each other in memory run on one XCD (slice_index), whose L2 then
//             reads every line from memory once.
//   passes    statistics by row chunks over the whole chip -> a small reduction -> the output pass: for slices that
//             do not fit and for batches with too few slices to fill the chip.
// Sums, statistics and gradients of w and b are f32; variances are combined from (count, mean, centred sum) triples,
// so a large mean costs no digits.  No atomics: sums have one order, results repeat bit for bit.
// Measured (bf16): forward 8 x 64 x 64 x 960 resident 34 us on an input that the 256 MB cache holds, 45 us (2.8 TB/s) on one
// that comes from memory; 16 x 64 x 64 x 320 33 us, 2.5 TB/s (4-byte loads: a vector divides ONE group's 20 bytes, also where
// a workgroup holds two); 8 x 8 x 1280 f32 4.8 us; one image of 64 x 64 x 320 by passes 17 us bf16, 13 us f32.
// Backward 8 x 64 x 64 x 960 by passes 80 us: sums 32 us at 3.9 TB/s, output 43 us at 4.4 TB/s, gradients of w and b 5 us;
// 2 x 16 x 16 x 640 resident 7.7 us + 2.5 us behind a forward of 5.2 us (one image: no second launch).
#include "sid_common.h"

#include <cstdint>

namespace {

constexpr int kXcd = 8;

template <int DT> struct Elem;
template <> struct Elem<SID_DTYPE_F32> { using type = float; };
template <> struct Elem<SID_DTYPE_BF16> { using type = __bf16; };
template <> struct Elem<SID_DTYPE_F16> { using type = _Float16; };

// VB bytes of memory held raw in registers
template <int VB> struct Raw { uint32_t w[VB / 4]; };
template <> struct Raw<2> { uint16_t w[1]; };

template <int VB>
__device__ __forceinline__ Raw<VB> load_raw(const char* p) {
    Raw<VB> r;
    if constexpr (VB == 2) r.w[0] = *(const uint16_t*)p;
    else if constexpr (VB == 4) r.w[0] = *(const uint32_t*)p;
    else if constexpr (VB == 8) { const uint2 v = *(const uint2*)p; r.w[0] = v.x; r.w[1] = v.y; }
    else { const uint4 v = *(const uint4*)p; r.w[0] = v.x; r.w[1] = v.y; r.w[2] = v.z; r.w[3] = v.w; }
    return r;
}

template <int VB>
__device__ __forceinline__ void store_raw(char* p, const Raw<VB>& r) {
    if constexpr (VB == 2) *(uint16_t*)p = r.w[0];
    else if constexpr (VB == 4) *(uint32_t*)p = r.w[0];
    else if constexpr (VB == 8) *(uint2*)p = make_uint2(r.w[0], r.w[1]);
    else *(uint4*)p = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
}

template <int DT, int VB>
__device__ __forceinline__ void unpack(const Raw<VB>& r, float* f) {
    constexpr int V = VB / (DT == SID_DTYPE_F32 ? 4 : 2);
    if constexpr (DT == SID_DTYPE_F32) {
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = __uint_as_float(r.w[e]);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const uint16_t h = VB == 2 ? (uint16_t)r.w[0] : (uint16_t)(r.w[e / 2] >> (16 * (e & 1)));
            if constexpr (DT == SID_DTYPE_BF16) f[e] = __uint_as_float((uint32_t)h << 16);
            else f[e] = (float)__builtin_bit_cast(_Float16, h);
        }
    }
}

template <int DT, int VB>
__device__ __forceinline__ Raw<VB> pack(const float* f) {
    constexpr int V = VB / (DT == SID_DTYPE_F32 ? 4 : 2);
    Raw<VB> r;
    if constexpr (DT == SID_DTYPE_F32) {
#pragma unroll
        for (int e = 0; e < V; ++e) r.w[e] = __float_as_uint(f[e]);
    } else {
        using T = typename Elem<DT>::type;
        uint16_t h[V];
#pragma unroll
        for (int e = 0; e < V; ++e) h[e] = __builtin_bit_cast(uint16_t, (T)f[e]);
        if constexpr (VB == 2) r.w[0] = h[0];
        else
#pragma unroll
            for (int e = 0; e < V; e += 2) r.w[e / 2] = (uint32_t)h[e] | ((uint32_t)h[e + 1] << 16);
    }
    return r;
}

__device__ __forceinline__ float sigmoid(float z) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.4426950408889634f));
}
// silu(z), and d silu / dz = s (1 + z (1 - s))
__device__ __forceinline__ float act_fwd(float z, int silu) { return silu ? z * sigmoid(z) : z; }
__device__ __forceinline__ float act_bwd(float z, float dy, int silu) {
    if (!silu) return dy;
    const float s = sigmoid(z);
    return dy * (s * (1.f + z * (1.f - s)));
}

// sum of K values over the workgroup, result in every thread; sm: K floats per wave
template <int K>
__device__ __forceinline__ void block_sum(float (&v)[K], float* sm) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) v[k] += __shfl_xor(v[k], off);
    const int wave = threadIdx.x >> 6, waves = (blockDim.x + 63) >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int k = 0; k < K; ++k) sm[wave * K + k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
        float s = 0.f;
        for (int w = 0; w < waves; ++w) s += sm[w * K + k];
        v[k] = s;
    }
}

// Sum of x over the threads of one of the workgroup's gc groups, in every thread of that group.
constexpr int kCluster = 4;
__device__ __forceinline__ void cluster_sum(float& x, int own, int gc, float* sm) {
    if (gc == 1) {
        float v[1] = {x};
        block_sum<1>(v, sm);
        x = v[0];
    } else {
        float v[kCluster];
#pragma unroll
        for (int k = 0; k < kCluster; ++k) v[k] = own == k ? x : 0.f;
        block_sum<kCluster>(v, sm);
#pragma unroll
        for (int k = 0; k < kCluster; ++k) x = own == k ? v[k] : x;
    }
}

// (n, mean, m2) <- (n, mean, m2) joined with (nb, meanb, m2b)
__device__ __forceinline__ void join(float& n, float& mean, float& m2, float nb, float meanb, float m2b) {
    const float t = n + nb;
    if (t > 0.f) {
        const float d = meanb - mean, f = nb / t;
        mean += d * f;
        m2 += m2b + d * d * (n * f);
        n = t;
    }
}

struct NormParams {
    const char *x, *dy;
    char* out;                    // y (forward) or dx (backward, or null)
    const float *w, *b;           // (C) or null: ones / zeros
    float *mean, *rstd;           // (B, G): written by the forward, read by the backward
    float2* part;                 // passes: [B][chunk][C]; resident backward: [B][C]
    float2* sums;                 // backward passes: [B][G] (s1, s2)
    float2* chan;                 // backward: [B][C] (dw, db) per image; null: one image, whose sums are the gradients
    float *dw, *db;               // (C), either may be null
    int B, N, C, G, Cg, silu, chunks, chunk_rows, out_rows;       // rows of a workgroup: statistics, output pass
    int gc;                       // resident forward: groups of one workgroup
    int fold;                     // passes: the output pass joins the chunks' group statistics itself
    float2* gpart;                // fold: [B][chunk][G]
    float eps;
};

// Work item of this workgroup when `items` of them follow each other in memory: workgroup i runs on XCD i mod 8, and
// every XCD takes one contiguous share.
__device__ __forceinline__ int slice_index(int items) {
    const int i = blockIdx.x, share = (items + kXcd - 1) / kXcd;
    return (i % kXcd) * share + i / kXcd;           // >= items for the tail: that workgroup has nothing to do
}

// ------------------------------------------------------------------------------------------------ resident
// Thread t < active owns vector column t mod cv of the group's cv vectors per row and rows t / cv + k rp: its
// channels never change, so w and b sit in registers.  NV vectors of VB bytes per thread.
template <int DT, int VB, int NV>
__global__ void __launch_bounds__(1024) gn_fwd_resident(NormParams p) {
    constexpr int ES = DT == SID_DTYPE_F32 ? 4 : 2, V = VB / ES;
    __shared__ float sm[16 * kCluster];
    const int per_image = p.G / p.gc, items = p.B * per_image, item = slice_index(items);
    if (item >= items) return;
    const int bi = item / per_image, g0 = (item - bi * per_image) * p.gc;
    const int cv = p.gc * p.Cg / V, rp = (int)blockDim.x / cv, t = threadIdx.x;
    const bool live = t < rp * cv;
    const int col = t % cv, row0 = t / cv, own = p.gc == 1 ? 0 : col * V / p.Cg;          // this thread's group of the gc
    const size_t pitch = (size_t)p.C * ES;
    const char* src = p.x + ((size_t)bi * p.N + row0) * pitch + ((size_t)g0 * p.Cg + (size_t)col * V) * ES;
    char* dst = p.out + (src - p.x);

    Raw<VB> raw[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k)
        if (live && row0 + k * rp < p.N) raw[k] = load_raw<VB>(src + (size_t)k * rp * pitch);
    const float inv_n = 1.f / ((float)p.N * (float)p.Cg);
    float s[1] = {0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k)
        if (live && row0 + k * rp < p.N) {
            float f[V];
            unpack<DT, VB>(raw[k], f);
#pragma unroll
            for (int e = 0; e < V; ++e) s[0] += f[e];
        }
    cluster_sum(s[0], own, p.gc, sm);
    const float mean = s[0] * inv_n;
    s[0] = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
        if (live && row0 + k * rp < p.N) {
            float f[V];
            unpack<DT, VB>(raw[k], f);
#pragma unroll
            for (int e = 0; e < V; ++e) { const float d = f[e] - mean; s[0] = __builtin_fmaf(d, d, s[0]); }
        }
    cluster_sum(s[0], own, p.gc, sm);
    const float rstd = 1.f / sqrtf(s[0] * inv_n + p.eps);
    if (!live) return;
    if (row0 == 0 && col * V == own * p.Cg) { p.mean[bi * p.G + g0 + own] = mean; p.rstd[bi * p.G + g0 + own] = rstd; }
    float w[V], b[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int c = g0 * p.Cg + col * V + e;
        w[e] = (p.w ? p.w[c] : 1.f) * rstd;
        b[e] = p.b ? p.b[c] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < NV; ++k)
        if (row0 + k * rp < p.N) {
            float f[V];
            unpack<DT, VB>(raw[k], f);
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] = act_fwd(__builtin_fmaf(f[e] - mean, w[e], b[e]), p.silu);
            store_raw<VB>(dst + (size_t)k * rp * pitch, pack<DT, VB>(f));
        }
}

template <int DT, int VB, int NV>
__global__ void __launch_bounds__(1024) gn_bwd_resident(NormParams p) {
    constexpr int ES = DT == SID_DTYPE_F32 ? 4 : 2, V = VB / ES;
    extern __shared__ float2 lds2[];                // [V][blockDim.x] per-thread channel sums
    __shared__ float sm[32];
    const int item = slice_index(p.B * p.G);
    if (item >= p.B * p.G) return;
    const int bi = item / p.G, g = item - bi * p.G;
    const int cv = p.Cg / V, rp = (int)blockDim.x / cv, t = threadIdx.x;
    const bool live = t < rp * cv;
    const int col = t % cv, row0 = t / cv;
    const size_t pitch = (size_t)p.C * ES;
    const size_t at = ((size_t)bi * p.N + row0) * pitch + ((size_t)g * p.Cg + (size_t)col * V) * ES;

    Raw<VB> rx[NV], rd[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k)
        if (live && row0 + k * rp < p.N) {
            rx[k] = load_raw<VB>(p.x + at + (size_t)k * rp * pitch);
            rd[k] = load_raw<VB>(p.dy + at + (size_t)k * rp * pitch);
        }
    const float mean = p.mean[item], rstd = p.rstd[item];
    float w[V], b[V], sw[V], sb[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int c = g * p.Cg + col * V + e;
        w[e] = live && p.w ? p.w[c] : 1.f;
        b[e] = live && p.b ? p.b[c] : 0.f;
        sw[e] = sb[e] = 0.f;
    }
#pragma unroll
    for (int k = 0; k < NV; ++k)
        if (live && row0 + k * rp < p.N) {
            float f[V], d[V];
            unpack<DT, VB>(rx[k], f);
            unpack<DT, VB>(rd[k], d);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float xh = (f[e] - mean) * rstd;
                const float dz = act_bwd(__builtin_fmaf(xh, w[e], b[e]), d[e], p.silu);
                sb[e] += dz;
                sw[e] = __builtin_fmaf(dz, xh, sw[e]);
            }
        }
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int e = 0; e < V; ++e) { s[0] = __builtin_fmaf(w[e], sb[e], s[0]); s[1] = __builtin_fmaf(w[e], sw[e], s[1]); }
    if (p.dw || p.db)
#pragma unroll
        for (int e = 0; e < V; ++e) lds2[e * blockDim.x + t] = make_float2(sw[e], sb[e]);
    block_sum<2>(s, sm);                            // its barriers also order the channel sums above
    const float inv_n = 1.f / ((float)p.N * (float)p.Cg);
    const float s1 = s[0] * inv_n, s2 = s[1] * inv_n;
    if (live && p.out)
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (row0 + k * rp < p.N) {
                float f[V], d[V];
                unpack<DT, VB>(rx[k], f);
                unpack<DT, VB>(rd[k], d);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float xh = (f[e] - mean) * rstd;
                    const float dz = act_bwd(__builtin_fmaf(xh, w[e], b[e]), d[e], p.silu);
                    f[e] = rstd * (__builtin_fmaf(dz, w[e], -s1) - xh * s2);
                }
                store_raw<VB>(p.out + at + (size_t)k * rp * pitch, pack<DT, VB>(f));
            }
    if (!p.dw && !p.db) return;
    // channel sums over the rp row threads, halving: thread t keeps the sums of rows t/cv, t/cv + h, ...
    for (int n = rp; n > 1;) {
        const int h = (n + 1) / 2;
        if (live && row0 + h < n && row0 < h)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float2 a = lds2[e * blockDim.x + t];
                const float2 c = lds2[e * blockDim.x + t + h * cv];
                a.x += c.x; a.y += c.y;
                lds2[e * blockDim.x + t] = a;
            }
        __syncthreads();
        n = h;
    }
    if (t < cv)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float2 a = lds2[e * blockDim.x + t];
            const int c = g * p.Cg + t * V + e;
            if (p.chan) {
                p.chan[(size_t)bi * p.C + c] = a;
            } else {
                if (p.dw) p.dw[c] = a.x;
                if (p.db) p.db[c] = a.y;
            }
        }
}

// ------------------------------------------------------------------------------------------------ passes
// Workgroups of 512 threads over (row chunk, image, slab of at most 512 vector columns).  Thread t < rp*cv owns vector
// column t mod cv of the slab and every rp-th row of the chunk.
struct Lane { int cv, rp, col, row, row_end; bool live; };
template <int V>
__device__ __forceinline__ Lane lane_of(const NormParams& p, int rows) {
    Lane l;
    const int cvs = p.C / V, slab0 = (int)blockIdx.z * 512;
    l.cv = min(512, cvs - slab0);
    l.rp = 512 / l.cv;
    const int t = threadIdx.x;
    l.live = t < l.rp * l.cv;
    l.col = slab0 + t % l.cv;
    const int r0 = (int)blockIdx.x * rows;
    l.row = r0 + t / l.cv;
    l.row_end = min(p.N, r0 + rows);
    return l;
}

constexpr int kFoldGroups = 512;
// Lanes that share one group's work in a workgroup of 512: a power of two, 64 at most.
__device__ __forceinline__ int lanes_per_group(int G) {
    int n = 64;
    while (n * G > 512) n >>= 1;
    return n;
}

template <int DT, int VB>
__global__ void __launch_bounds__(512) gn_stats(NormParams p) {
    constexpr int ES = DT == SID_DTYPE_F32 ? 4 : 2, V = VB / ES, R = 8;
    __shared__ float lm[V][512], l2[V][512], ln[512];
    const Lane l = lane_of<V>(p, p.chunk_rows);
    const size_t pitch = (size_t)p.C * ES;
    const char* src = p.x + (size_t)blockIdx.y * p.N * pitch + (size_t)l.col * VB;
    float n = 0.f, mean[V], m2[V];
#pragma unroll
    for (int e = 0; e < V; ++e) mean[e] = m2[e] = 0.f;
    // batches of R rows: their mean, then their centred sum, from registers
    for (int r = l.row; l.live && r < l.row_end; r += R * l.rp) {
        Raw<VB> raw[R];
        float cnt = 0.f, s[V], q[V];
#pragma unroll
        for (int k = 0; k < R; ++k)
            if (r + k * l.rp < l.row_end) raw[k] = load_raw<VB>(src + (size_t)(r + k * l.rp) * pitch);
#pragma unroll
        for (int e = 0; e < V; ++e) s[e] = q[e] = 0.f;
#pragma unroll
        for (int k = 0; k < R; ++k)
            if (r + k * l.rp < l.row_end) {
                float f[V];
                unpack<DT, VB>(raw[k], f);
                cnt += 1.f;
#pragma unroll
                for (int e = 0; e < V; ++e) s[e] += f[e];
            }
        const float ic = 1.f / cnt;
#pragma unroll
        for (int e = 0; e < V; ++e) s[e] *= ic;
#pragma unroll
        for (int k = 0; k < R; ++k)
            if (r + k * l.rp < l.row_end) {
                float f[V];
                unpack<DT, VB>(raw[k], f);
#pragma unroll
                for (int e = 0; e < V; ++e) { const float d = f[e] - s[e]; q[e] = __builtin_fmaf(d, d, q[e]); }
            }
        const float tot = n + cnt, fr = cnt / tot, nf = n * fr;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float d = s[e] - mean[e];
            mean[e] += d * fr;
            m2[e] += q[e] + d * d * nf;
        }
        n = tot;
    }
    const int t = threadIdx.x;
    ln[t] = n;
#pragma unroll
    for (int e = 0; e < V; ++e) { lm[e][t] = mean[e]; l2[e][t] = m2[e]; }
    __syncthreads();
    const int rt = t / l.cv;
    for (int m = l.rp; m > 1;) {
        const int h = (m + 1) / 2;
        if (l.live && rt < h && rt + h < m) {
            const int o = t + h * l.cv;
            const float nb = ln[o];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float na = n;
                join(na, mean[e], m2[e], nb, lm[e][o], l2[e][o]);
                lm[e][t] = mean[e];
                l2[e][t] = m2[e];
            }
            n += nb;
            ln[t] = n;
        }
        __syncthreads();
        m = h;
    }
    if (t < l.cv) {
        float2* out = p.part + ((size_t)blockIdx.y * p.chunks + blockIdx.x) * p.C + (size_t)l.col * V;
#pragma unroll
        for (int e = 0; e < V; ++e) out[e] = make_float2(mean[e], m2[e]);
    }
}

// Sums over the rp row threads and Cg channels of group g of what ls holds per thread and channel; in the L lanes of the group.
template <int V>
__device__ __forceinline__ float group_sum(const float (&ls)[V][512], const NormParams& p, const Lane& l, int g, int lane, int L) {
    float s = 0.f;
    if (g < p.G)
        for (int i = lane; i < p.Cg; i += L) {
            const int c = g * p.Cg + i;
            const float* at = &ls[c % V][c / V];
            for (int r = 0; r < l.rp; ++r) s += at[r * l.cv];
        }
    for (int off = L >> 1; off >= 1; off >>= 1) s += __shfl_xor(s, off);
    return s;
}

// fold: (mean, centred sum) per group and chunk.  A batch of rows sits in registers: the group's mean over the workgroup,
// then the sum of squares about it; batches join by their counts.
template <int DT, int VB>
__global__ void __launch_bounds__(512) gn_group_stats(NormParams p) {
    constexpr int ES = DT == SID_DTYPE_F32 ? 4 : 2, V = VB / ES, R = 8;
    __shared__ float ls[V][512], gm[kFoldGroups];
    const Lane l = lane_of<V>(p, p.chunk_rows);
    const int t = threadIdx.x, L = lanes_per_group(p.G), g = t / L, lane = t % L;
    const size_t pitch = (size_t)p.C * ES;
    const char* src = p.x + (size_t)blockIdx.y * p.N * pitch + (size_t)l.col * VB;
    float n = 0.f, mean = 0.f, m2 = 0.f;
    int of[V];                       // groups of this thread's channels
#pragma unroll
    for (int e = 0; e < V; ++e) of[e] = (l.col * V + e) / p.Cg;
    for (int r0 = (int)blockIdx.x * p.chunk_rows; r0 < l.row_end; r0 += R * l.rp) {
        const int row = r0 + t / l.cv;
        Raw<VB> raw[R];
#pragma unroll
        for (int k = 0; k < R; ++k) raw[k] = load_raw<VB>(src + (size_t)min(row + k * l.rp, l.row_end - 1) * pitch);
        float s[V];
#pragma unroll
        for (int e = 0; e < V; ++e) s[e] = 0.f;
#pragma unroll
        for (int k = 0; k < R; ++k)
            if (l.live && row + k * l.rp < l.row_end) {
                float f[V];
                unpack<DT, VB>(raw[k], f);
#pragma unroll
                for (int e = 0; e < V; ++e) s[e] += f[e];
            }
#pragma unroll
        for (int e = 0; e < V; ++e) ls[e][t] = s[e];
        __syncthreads();
        const float count = (float)min(l.row_end - r0, R * l.rp) * (float)p.Cg;
        const float bm = group_sum<V>(ls, p, l, g, lane, L) / count;
        if (g < p.G && lane == 0) gm[g] = bm;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float m = gm[of[e]];
            float q = 0.f;
#pragma unroll
            for (int k = 0; k < R; ++k)
                if (l.live && row + k * l.rp < l.row_end) {
                    float f[V];
                    unpack<DT, VB>(raw[k], f);
                    const float d = f[e] - m;
                    q = __builtin_fmaf(d, d, q);
                }
            ls[e][t] = q;
        }
        __syncthreads();
        join(n, mean, m2, count, bm, group_sum<V>(ls, p, l, g, lane, L));
        __syncthreads();
    }
    if (g < p.G && lane == 0) p.gpart[((size_t)blockIdx.y * p.chunks + blockIdx.x) * p.G + g] = make_float2(mean, m2);
}

// Joins (n, mean, m2) over the `width` lanes that share a group; the same bits in all of them.
__device__ __forceinline__ void join_lanes(float& n, float& mean, float& m2, int width) {
    for (int off = width >> 1; off >= 1; off >>= 1) {
        const float nb = __shfl_xor(n, off), mb = __shfl_xor(mean, off), qb = __shfl_xor(m2, off);
        if (threadIdx.x & off) { float a = nb, b = mb, c = qb; join(a, b, c, n, mean, m2); n = a; mean = b; m2 = c; }
        else join(n, mean, m2, nb, mb, qb);
    }
}

// One workgroup per (image, group): joins chunks x Cg triples into mean and rstd.
__global__ void __launch_bounds__(256) gn_join(NormParams p) {
    __shared__ float sn[4], sm[4], s2[4];
    const int bi = blockIdx.x / p.G, g = blockIdx.x - bi * p.G;
    float n = 0.f, mean = 0.f, m2 = 0.f;
    const int total = p.chunks * p.Cg;
    for (int i = threadIdx.x; i < total; i += 256) {
        const int ch = i / p.Cg, c = i - ch * p.Cg;
        const float2 v = p.part[((size_t)bi * p.chunks + ch) * p.C + (size_t)g * p.Cg + c];
        join(n, mean, m2, (float)min(p.chunk_rows, p.N - ch * p.chunk_rows), v.x, v.y);
    }
    join_lanes(n, mean, m2, 64);
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) { sn[wave] = n; sm[wave] = mean; s2[wave] = m2; }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 4; ++w) join(n, mean, m2, sn[w], sm[w], s2[w]);
        p.mean[blockIdx.x] = mean;
        p.rstd[blockIdx.x] = 1.f / sqrtf(m2 / ((float)p.N * (float)p.Cg) + p.eps);
    }
}

template <int DT, int VB>
__global__ void __launch_bounds__(512) gn_apply(NormParams p) {
    constexpr int ES = DT == SID_DTYPE_F32 ? 4 : 2, V = VB / ES, R = 4;
    __shared__ float2 st[kFoldGroups];
    const Lane l = lane_of<V>(p, p.out_rows);
    if (p.fold) {
        const int L = lanes_per_group(p.G), g = (int)threadIdx.x / L, lane = (int)threadIdx.x % L;
        // the mean of the chunks' means by their rows, then the centred sums about it
        const float2* part = p.gpart + (size_t)blockIdx.y * p.chunks * p.G + (g < p.G ? g : 0);
        float mean = 0.f, m2 = 0.f;
#pragma unroll 4
        for (int ch = lane; ch < p.chunks; ch += L)
            mean = __builtin_fmaf((float)min(p.chunk_rows, p.N - ch * p.chunk_rows), part[(size_t)ch * p.G].x, mean);
        for (int off = L >> 1; off >= 1; off >>= 1) mean += __shfl_xor(mean, off);
        mean /= (float)p.N;
#pragma unroll 4
        for (int ch = lane; ch < p.chunks; ch += L) {
            const float2 v = part[(size_t)ch * p.G];
            const float d = v.x - mean;
            m2 += __builtin_fmaf((float)min(p.chunk_rows, p.N - ch * p.chunk_rows) * (float)p.Cg, d * d, v.y);
        }
        for (int off = L >> 1; off >= 1; off >>= 1) m2 += __shfl_xor(m2, off);
        if (g < p.G && lane == 0) {
            const float rstd = 1.f / sqrtf(m2 / ((float)p.N * (float)p.Cg) + p.eps);
            st[g] = make_float2(mean, rstd);
            if (blockIdx.x == 0) { p.mean[blockIdx.y * p.G + g] = mean; p.rstd[blockIdx.y * p.G + g] = rstd; }
        }
        __syncthreads();
    }
    if (!l.live) return;
    const size_t pitch = (size_t)p.C * ES, base = (size_t)blockIdx.y * p.N * pitch + (size_t)l.col * VB;
    float mean[V], w[V], b[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int c = l.col * V + e, gi = (int)blockIdx.y * p.G + c / p.Cg;
        mean[e] = p.fold ? st[c / p.Cg].x : p.mean[gi];
        w[e] = (p.w ? p.w[c] : 1.f) * (p.fold ? st[c / p.Cg].y : p.rstd[gi]);
        b[e] = p.b ? p.b[c] : 0.f;
    }
    for (int r = l.row; r < l.row_end; r += R * l.rp) {
        Raw<VB> raw[R];
#pragma unroll
        for (int k = 0; k < R; ++k)
            if (r + k * l.rp < l.row_end) raw[k] = load_raw<VB>(p.x + base + (size_t)(r + k * l.rp) * pitch);
#pragma unroll
        for (int k = 0; k < R; ++k)
            if (r + k * l.rp < l.row_end) {
                float f[V];
                unpack<DT, VB>(raw[k], f);
#pragma unroll
                for (int e = 0; e < V; ++e) f[e] = act_fwd(__builtin_fmaf(f[e] - mean[e], w[e], b[e]), p.silu);
                store_raw<VB>(p.out + base + (size_t)(r + k * l.rp) * pitch, pack<DT, VB>(f));
            }
    }
}

// Per channel and chunk: (sum dz xh, sum dz)
template <int DT, int VB>
__global__ void __launch_bounds__(512) gn_bwd_sums(NormParams p) {
    constexpr int ES = DT == SID_DTYPE_F32 ? 4 : 2, V = VB / ES, R = 4;
    __shared__ float2 ls[V][512];
    const Lane l = lane_of<V>(p, p.chunk_rows);
    const size_t pitch = (size_t)p.C * ES, base = (size_t)blockIdx.y * p.N * pitch + (size_t)l.col * VB;
    float mean[V], rstd[V], w[V], b[V], sw[V], sb[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int c = l.live ? l.col * V + e : 0, gi = (int)blockIdx.y * p.G + c / p.Cg;
        mean[e] = p.mean[gi];
        rstd[e] = p.rstd[gi];
        w[e] = p.w ? p.w[c] : 1.f;
        b[e] = p.b ? p.b[c] : 0.f;
        sw[e] = sb[e] = 0.f;
    }
    for (int r = l.row; l.live && r < l.row_end; r += R * l.rp) {
        Raw<VB> rx[R], rd[R];
#pragma unroll
        for (int k = 0; k < R; ++k)
            if (r + k * l.rp < l.row_end) {
                rx[k] = load_raw<VB>(p.x + base + (size_t)(r + k * l.rp) * pitch);
                rd[k] = load_raw<VB>(p.dy + base + (size_t)(r + k * l.rp) * pitch);
            }
#pragma unroll
        for (int k = 0; k < R; ++k)
            if (r + k * l.rp < l.row_end) {
                float f[V], d[V];
                unpack<DT, VB>(rx[k], f);
                unpack<DT, VB>(rd[k], d);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float xh = (f[e] - mean[e]) * rstd[e];
                    const float dz = act_bwd(__builtin_fmaf(xh, w[e], b[e]), d[e], p.silu);
                    sb[e] += dz;
                    sw[e] = __builtin_fmaf(dz, xh, sw[e]);
                }
            }
    }
    const int t = threadIdx.x, rt = t / l.cv;
#pragma unroll
    for (int e = 0; e < V; ++e) ls[e][t] = make_float2(sw[e], sb[e]);
    __syncthreads();
    for (int m = l.rp; m > 1;) {
        const int h = (m + 1) / 2;
        if (l.live && rt < h && rt + h < m)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float2 c = ls[e][t + h * l.cv];
                sw[e] += c.x; sb[e] += c.y;
                ls[e][t] = make_float2(sw[e], sb[e]);
            }
        __syncthreads();
        m = h;
    }
    if (t < l.cv) {
        float2* out = p.part + ((size_t)blockIdx.y * p.chunks + blockIdx.x) * p.C + (size_t)l.col * V;
#pragma unroll
        for (int e = 0; e < V; ++e) out[e] = make_float2(sw[e], sb[e]);
    }
    if (p.fold) {
        const int L = lanes_per_group(p.G), g = t / L, lane = t % L;
        float s1 = 0.f, s2 = 0.f;
        if (g < p.G)
            for (int c = lane; c < p.Cg; c += L) {
                const int cc = g * p.Cg + c;
                const float wc = p.w ? p.w[cc] : 1.f;
                const float2 v = ls[cc % V][cc / V];
                s1 = __builtin_fmaf(wc, v.y, s1);
                s2 = __builtin_fmaf(wc, v.x, s2);
            }
        for (int off = L >> 1; off >= 1; off >>= 1) { s1 += __shfl_xor(s1, off); s2 += __shfl_xor(s2, off); }
        if (g < p.G && lane == 0) p.gpart[((size_t)blockIdx.y * p.chunks + blockIdx.x) * p.G + g] = make_float2(s1, s2);
    }
}

// One workgroup per (image, group): channel sums over the chunks, then the group's s1 and s2.
__global__ void __launch_bounds__(256) gn_bwd_join(NormParams p) {
    __shared__ float2 ls[256];
    __shared__ float sm[8];
    const int bi = blockIdx.x / p.G, g = blockIdx.x - bi * p.G, t = threadIdx.x;
    const int cols = min(p.Cg, 256), rp = 256 / cols, rt = t / cols;
    float s[2] = {0.f, 0.f};
    for (int c0 = 0; c0 < p.Cg; c0 += cols) {
        const int c = c0 + t % cols;
        const bool live = t < rp * cols && c < p.Cg;
        float2 a = make_float2(0.f, 0.f);
        if (live)
            for (int ch = rt; ch < p.chunks; ch += rp) {
                const float2 v = p.part[((size_t)bi * p.chunks + ch) * p.C + (size_t)g * p.Cg + c];
                a.x += v.x; a.y += v.y;
            }
        __syncthreads();
        ls[t] = a;
        __syncthreads();
        for (int m = rp; m > 1;) {
            const int h = (m + 1) / 2;
            if (live && rt < h && rt + h < m) {
                const float2 o = ls[t + h * cols];
                a.x += o.x; a.y += o.y;
                ls[t] = a;
            }
            __syncthreads();
            m = h;
        }
        if (live && rt == 0) {
            const int cc = g * p.Cg + c;
            if (p.chan) p.chan[(size_t)bi * p.C + cc] = a;
            const float w = p.w ? p.w[cc] : 1.f;
            s[0] = __builtin_fmaf(w, a.y, s[0]);
            s[1] = __builtin_fmaf(w, a.x, s[1]);
        }
    }
    block_sum<2>(s, sm);
    const float inv_n = 1.f / ((float)p.N * (float)p.Cg);
    if (t == 0) p.sums[blockIdx.x] = make_float2(s[0] * inv_n, s[1] * inv_n);
}

template <int DT, int VB>
__global__ void __launch_bounds__(512) gn_bwd_apply(NormParams p) {
    constexpr int ES = DT == SID_DTYPE_F32 ? 4 : 2, V = VB / ES, R = 4;
    __shared__ float2 st[kFoldGroups];
    const Lane l = lane_of<V>(p, p.out_rows);
    if (p.fold) {
        const int L = lanes_per_group(p.G), g = (int)threadIdx.x / L, lane = (int)threadIdx.x % L;
        float a = 0.f, c = 0.f;
        if (g < p.G)
#pragma unroll 4
            for (int ch = lane; ch < p.chunks; ch += L) {
                const float2 v = p.gpart[((size_t)blockIdx.y * p.chunks + ch) * p.G + g];
                a += v.x; c += v.y;
            }
        for (int off = L >> 1; off >= 1; off >>= 1) { a += __shfl_xor(a, off); c += __shfl_xor(c, off); }
        const float inv_n = 1.f / ((float)p.N * (float)p.Cg);
        if (g < p.G && lane == 0) st[g] = make_float2(a * inv_n, c * inv_n);
        __syncthreads();
    }
    if (!l.live) return;
    const size_t pitch = (size_t)p.C * ES, base = (size_t)blockIdx.y * p.N * pitch + (size_t)l.col * VB;
    float mean[V], rstd[V], w[V], b[V], s1[V], s2[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int c = l.col * V + e, gi = (int)blockIdx.y * p.G + c / p.Cg;
        mean[e] = p.mean[gi];
        rstd[e] = p.rstd[gi];
        w[e] = p.w ? p.w[c] : 1.f;
        b[e] = p.b ? p.b[c] : 0.f;
        const float2 s = p.fold ? st[c / p.Cg] : p.sums[gi];
        s1[e] = s.x; s2[e] = s.y;
    }
    for (int r = l.row; r < l.row_end; r += R * l.rp) {
        Raw<VB> rx[R], rd[R];
#pragma unroll
        for (int k = 0; k < R; ++k)
            if (r + k * l.rp < l.row_end) {
                rx[k] = load_raw<VB>(p.x + base + (size_t)(r + k * l.rp) * pitch);
                rd[k] = load_raw<VB>(p.dy + base + (size_t)(r + k * l.rp) * pitch);
            }
#pragma unroll
        for (int k = 0; k < R; ++k)
            if (r + k * l.rp < l.row_end) {
                float f[V], d[V];
                unpack<DT, VB>(rx[k], f);
                unpack<DT, VB>(rd[k], d);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float xh = (f[e] - mean[e]) * rstd[e];
                    const float dz = act_bwd(__builtin_fmaf(xh, w[e], b[e]), d[e], p.silu);
                    f[e] = rstd[e] * (__builtin_fmaf(dz, w[e], -s1[e]) - xh * s2[e]);
                }
                store_raw<VB>(p.out + base + (size_t)(r + k * l.rp) * pitch, pack<DT, VB>(f));
            }
    }
}

// dw, db: `rows` rows of channel sums (images, or images x chunks), 32 channels a workgroup, every 32nd row a thread, then
// the 32 threads of a channel in halves.
__global__ void __launch_bounds__(1024) gn_param_grads(const float2* rows_of, float* dw, float* db, int rows, int C) {
    __shared__ float2 ls[1024];
    const int t = threadIdx.x, c = blockIdx.x * 32 + (t & 31), r0 = t >> 5;
    float sw = 0.f, sb = 0.f;
    if (c < C)
#pragma unroll 8
        for (int r = r0; r < rows; r += 32) {
            const float2 v = rows_of[(size_t)r * C + c];
            sw += v.x; sb += v.y;
        }
    ls[t] = make_float2(sw, sb);
    __syncthreads();
    for (int h = 16; h >= 1; h >>= 1) {
        if (r0 < h) {
            const float2 o = ls[t + h * 32];
            sw += o.x; sb += o.y;
            ls[t] = make_float2(sw, sb);
        }
        __syncthreads();
    }
    if (r0 == 0 && c < C) {
        if (dw) dw[c] = sw;
        if (db) db[c] = sb;
    }
}

// ------------------------------------------------------------------------------------------------ host
struct Plan {
    int vb;            // bytes of one vector
    int nv;            // resident: class of vectors per thread (bytes / vb), 0 = passes
    int threads;       // resident
    int gc;            // resident forward: groups of one workgroup
    int chunks, chunk_rows, out_rows, fold;
    size_t part_bytes, sums_bytes, chan_bytes;
};

int vec_bytes(long long span, uintptr_t addr, int es) {
    for (int vb = 16; vb > es; vb /= 2)
        if (span % vb == 0 && addr % vb == 0) return vb;
    return es;
}

// Registers in which a thread of the resident form may hold its slice, by class: 1024 threads leave 128 each, so the
// forward keeps up to 64 of x, the backward up to 24 of x and 24 of dy.
constexpr int kFwdRegs[3] = {8, 24, 64}, kBwdRegs[2] = {8, 24};
constexpr int vectors_in(int regs, int vb) { return vb >= 4 ? regs * 4 / vb : regs; }

Plan make_plan(int B, int N, int C, int G, int dtype, uintptr_t addr, bool bwd) {
    const int es = dtype == SID_DTYPE_F32 ? 4 : 2, Cg = C / G;
    Plan pl{};
    const int vb = vec_bytes((long long)Cg * es, addr, es), cv = Cg * es / vb;
    // Slices above 64 KB go by passes where the resident kernel's few workgroups would read them alone (forward, bf16: 64 x 64 x
    // 320 of one image 20.5 us resident, 17.2 in passes; of four, 18.7 and 26.9) and always backward, where a thread holds two
    // tensors (64 x 64 x 320 of sixteen images: 74 us resident, 60 in passes; of one, 36 and 24), and with an odd number of 16-bit
    // channels a group, whose pieces only go two bytes at a time (64 x 64 x 480 of sixteen images: 69 and 45).
    const bool large = (size_t)N * Cg * es > (64u << 10);
    if (cv <= 1024 && !(large && (bwd || vb == 2 || (long long)B * G <= 64))) {
        for (int threads = 256; threads <= 1024 && !pl.nv; threads *= 2) {
            if (cv > threads) continue;
            const int rows = (N + threads / cv - 1) / (threads / cv);
            const int* regs = bwd ? kBwdRegs : kFwdRegs;
            // a workgroup of 256 or 512 threads only while a thread holds little: more threads hide more latency
            const int last = threads < 1024 ? 1 : bwd ? 2 : 3;
            for (int i = 0; i < last; ++i)
                if (rows <= vectors_in(regs[i], vb)) { pl.nv = vectors_in(regs[i], vb); pl.threads = threads; break; }
        }
    }
    pl.vb = vb;
    pl.gc = 1;
    if (!bwd && pl.nv) {
        // Neighbouring groups in one workgroup while a row's piece is below a cache line, the slice still fits, there are
        // workgroups for every CU and enough rows: a piece costs an L2 request whatever its length, a workgroup of several
        // groups has twice the threads to bring together (16 images of 320 channels, one group and two: 64 x 64 34.2 and 31.8 us,
        // 48 x 48 20.7 both, 32 x 32 11.5 and 14.9, 16 x 16 5.6 and 9.4).
        for (int gc = 2; gc <= kCluster && G % gc == 0 && N >= 2560 && (long long)B * G / gc >= 256 && gc * cv <= 1024 && gc * Cg * es <= 128; gc *= 2) {
            const int rows = (N + 1024 / (gc * cv) - 1) / (1024 / (gc * cv));
            for (int i = 0; i < 3; ++i)
                if (rows <= vectors_in(kFwdRegs[i], vb)) { pl.gc = gc; pl.threads = 1024; pl.nv = vectors_in(kFwdRegs[i], vb); break; }
        }
    }
    if (pl.nv) {
        // one image's sums are the gradients: a launch less (16 x 16 x 640 forward and backward 12.9 -> 11.6 us).  Walking two
        // images in one workgroup to the same end costs more than the launch (13.1 -> 14.3 us; 2 x 32 x 32 x 320 18 -> 28 us).
        pl.chan_bytes = bwd && B > 1 ? (size_t)B * C * sizeof(float2) : 0;
        return pl;
    }
    pl.vb = vec_bytes((long long)C * es, addr, es);
    // Chunks: two workgroups of 512 threads for every CU, and two rows or more for every thread.  Every workgroup of the output
    // pass joins the group statistics of its image's chunks itself, so these are 128 at most; where a row takes several
    // workgroups, or there are more groups than threads, a launch of its own joins them.
    const int cvs = C * es / pl.vb, slabs = (cvs + 511) / 512, rp = 512 / (cvs < 512 ? cvs : 512);
    pl.fold = slabs == 1 && G <= kFoldGroups;
    long long want = 512 / ((long long)B * slabs);
    if (want < 1) want = 1;
    if (pl.fold && want > 128) want = 128;
    long long rows = (N + want - 1) / want;
    if (rows < 2 * rp) rows = 2 * rp;
    if (rows > N) rows = N;
    pl.chunk_rows = (int)rows;
    pl.chunks = (int)((N + rows - 1) / rows);
    // the output pass keeps no sums: more, smaller workgroups
    const long long out = 1024 / ((long long)B * slabs);
    long long orows = (N + (out < 1 ? 1 : out) - 1) / (out < 1 ? 1 : out);
    if (orows < 4 * rp) orows = 4 * rp;
    pl.out_rows = (int)(orows > N ? N : orows);
    pl.part_bytes = pl.fold && !bwd ? 0 : sid::align_up((size_t)B * pl.chunks * C * sizeof(float2), 256);
    pl.sums_bytes = pl.fold ? sid::align_up((size_t)B * pl.chunks * G * sizeof(float2), 256) : bwd ? sid::align_up((size_t)B * G * sizeof(float2), 256) : 0;
    pl.chan_bytes = bwd && !pl.fold ? (size_t)B * C * sizeof(float2) : 0;
    return pl;
}

size_t plan_bytes(const Plan& pl) { return pl.part_bytes + pl.sums_bytes + pl.chan_bytes; }

// A launch holds fewer than 2^32 threads in x and 2^16 workgroups in z.
int check_launch(const Plan& pl, int B, int C, int G, int dtype) {
    const long long items = (long long)B * (G / pl.gc) + kXcd;                    // resident workgroups, or those of a join
    const long long slabs = ((long long)C * (dtype == SID_DTYPE_F32 ? 4 : 2) / pl.vb + 511) / 512;
    const bool fits = pl.nv ? items * pl.threads < (1LL << 32) : slabs < (1 << 16) && (pl.fold || items * 256 < (1LL << 32));
    SID_CHECK_ARG(fits && C <= (1 << 27) - 32, "tensor too large: %d channels, %lld groups", C, (long long)B * G);      // 32 threads a channel
    return SID_OK;
}

int check_shape(int B, int N, int C, int G, int dtype) {
    SID_CHECK_ARG(B >= 1 && N >= 1 && C >= 1 && G >= 1, "B, N, C, G must be >= 1");
    SID_CHECK_ARG(C % G == 0, "%d channels do not divide into %d groups", C, G);
    SID_CHECK_ARG(dtype == SID_DTYPE_F32 || dtype == SID_DTYPE_BF16 || dtype == SID_DTYPE_F16, "unknown dtype %d", dtype);
    // rows are 32-bit integers, and the passes count up to 8 rows of 512 threads and a chunk's rounding (2048 rows at most) past N
    SID_CHECK_ARG((long long)B * N * C < (1LL << 40) && (long long)N * (C / G) < (1LL << 31) - (1 << 16) && (long long)B * C < (1LL << 31) &&
                  (long long)B * G < (1 << 30) && B < 65536, "tensor too large");
    return SID_OK;
}

bool aligned_to_elements(uintptr_t addr, int dtype) { return addr % (dtype == SID_DTYPE_F32 ? 4 : 2) == 0; }

template <int DT, int VB>
int launch_fwd(const NormParams& p, const Plan& pl, hipStream_t st) {
    if (pl.nv) {
        const int items = p.B * (p.G / p.gc);
        const dim3 grid((items + kXcd - 1) / kXcd * kXcd), block(pl.threads);
        if (pl.nv == vectors_in(kFwdRegs[0], VB)) hipLaunchKernelGGL((gn_fwd_resident<DT, VB, vectors_in(kFwdRegs[0], VB)>), grid, block, 0, st, p);
        else if (pl.nv == vectors_in(kFwdRegs[1], VB)) hipLaunchKernelGGL((gn_fwd_resident<DT, VB, vectors_in(kFwdRegs[1], VB)>), grid, block, 0, st, p);
        else hipLaunchKernelGGL((gn_fwd_resident<DT, VB, vectors_in(kFwdRegs[2], VB)>), grid, block, 0, st, p);
    } else {
        const int cvs = p.C / (VB / (DT == SID_DTYPE_F32 ? 4 : 2));
        const dim3 grid(pl.chunks, p.B, (cvs + 511) / 512), out((p.N + p.out_rows - 1) / p.out_rows, p.B, (cvs + 511) / 512);
        if (p.fold) {
            hipLaunchKernelGGL((gn_group_stats<DT, VB>), grid, dim3(512), 0, st, p);
        } else {
            hipLaunchKernelGGL((gn_stats<DT, VB>), grid, dim3(512), 0, st, p);
            hipLaunchKernelGGL(gn_join, dim3(p.B * p.G), dim3(256), 0, st, p);
        }
        hipLaunchKernelGGL((gn_apply<DT, VB>), out, dim3(512), 0, st, p);
    }
    SID_CHECK_HIP(hipGetLastError());
    return SID_OK;
}

template <int DT, int VB>
int launch_bwd(const NormParams& p, const Plan& pl, hipStream_t st) {
    if (pl.nv) {
        const dim3 grid(((p.B * p.G + kXcd - 1) / kXcd) * kXcd), block(pl.threads);
        const size_t lds = p.dw || p.db ? (size_t)pl.threads * (VB / (DT == SID_DTYPE_F32 ? 4 : 2)) * sizeof(float2) : 0;
        if (pl.nv == vectors_in(kBwdRegs[0], VB)) {
            int rc = sid::allow_dynamic_lds<gn_bwd_resident<DT, VB, vectors_in(kBwdRegs[0], VB)>>(65536);
            if (rc) return rc;
            hipLaunchKernelGGL((gn_bwd_resident<DT, VB, vectors_in(kBwdRegs[0], VB)>), grid, block, lds, st, p);
        } else {
            int rc = sid::allow_dynamic_lds<gn_bwd_resident<DT, VB, vectors_in(kBwdRegs[1], VB)>>(65536);
            if (rc) return rc;
            hipLaunchKernelGGL((gn_bwd_resident<DT, VB, vectors_in(kBwdRegs[1], VB)>), grid, block, lds, st, p);
        }
    } else {
        const int cvs = p.C / (VB / (DT == SID_DTYPE_F32 ? 4 : 2));
        const dim3 grid(pl.chunks, p.B, (cvs + 511) / 512), out((p.N + p.out_rows - 1) / p.out_rows, p.B, (cvs + 511) / 512);
        hipLaunchKernelGGL((gn_bwd_sums<DT, VB>), grid, dim3(512), 0, st, p);
        if (!p.fold) hipLaunchKernelGGL(gn_bwd_join, dim3(p.B * p.G), dim3(256), 0, st, p);
        if (p.out) hipLaunchKernelGGL((gn_bwd_apply<DT, VB>), out, dim3(512), 0, st, p);
    }
    if ((p.dw || p.db) && !(pl.nv && p.B == 1)) {
        const bool chunks = !pl.nv && p.fold;            // the chunks' sums themselves
        hipLaunchKernelGGL(gn_param_grads, dim3((p.C + 31) / 32), dim3(1024), 0, st, chunks ? p.part : p.chan, p.dw, p.db,
                           chunks ? p.B * p.chunks : p.B, p.C);
    }
    SID_CHECK_HIP(hipGetLastError());
    return SID_OK;
}

template <int DT>
int by_vec(const NormParams& p, const Plan& pl, bool bwd, hipStream_t st) {
    switch (pl.vb) {
        case 16: return bwd ? launch_bwd<DT, 16>(p, pl, st) : launch_fwd<DT, 16>(p, pl, st);
        case 8: return bwd ? launch_bwd<DT, 8>(p, pl, st) : launch_fwd<DT, 8>(p, pl, st);
        case 4: return bwd ? launch_bwd<DT, 4>(p, pl, st) : launch_fwd<DT, 4>(p, pl, st);
        default:
            if constexpr (DT != SID_DTYPE_F32) return bwd ? launch_bwd<DT, 2>(p, pl, st) : launch_fwd<DT, 2>(p, pl, st);
            return sid::fail(SID_EINVAL, "tensors must be aligned to their element size");
    }
}

int by_dtype(const NormParams& p, const Plan& pl, int dtype, bool bwd, hipStream_t st) {
    if (dtype == SID_DTYPE_F32) return by_vec<SID_DTYPE_F32>(p, pl, bwd, st);
    if (dtype == SID_DTYPE_BF16) return by_vec<SID_DTYPE_BF16>(p, pl, bwd, st);
    return by_vec<SID_DTYPE_F16>(p, pl, bwd, st);
}

NormParams params_of(int B, int N, int C, int G, int act) {
    NormParams p{};
    p.B = B; p.N = N; p.C = C; p.G = G; p.Cg = C / G;
    p.silu = act == SID_ACT_SILU;
    return p;
}

}  // namespace

extern "C" size_t sid_group_norm_workspace_bytes(int B, int N, int C, int G, int dtype, int backward) {
    if (check_shape(B, N, C, G, dtype)) return 0;
    // whatever the tensors' alignment: the vector width decides between the forms
    size_t most = 256;
    for (uintptr_t addr = 16; addr >= 2; addr /= 2) {
        const size_t n = plan_bytes(make_plan(B, N, C, G, dtype, addr, backward != 0));
        most = n > most ? n : most;
    }
    return most;
}

extern "C" int sid_group_norm_plan(int B, int N, int C, int G, int dtype, int backward, int plan[6]) {
    SID_CHECK_ARG(plan, "NULL pointer");
    if (int rc = check_shape(B, N, C, G, dtype)) return rc;
    const Plan pl = make_plan(B, N, C, G, dtype, 0, backward != 0);
    plan[0] = pl.nv; plan[1] = pl.vb; plan[2] = pl.nv ? pl.threads : 512; plan[3] = pl.gc; plan[4] = pl.chunks; plan[5] = pl.fold;
    return SID_OK;
}

extern "C" int sid_group_norm_act_fwd(const void* x, const float* weight, const float* bias, void* y, float* mean, float* rstd,
                                      int B, int N, int C, int G, float eps, int act, int dtype,
                                      void* workspace, size_t workspace_bytes, void* stream) {
    SID_CHECK_ARG(x && y && mean && rstd, "NULL tensor pointer");
    if (int rc = check_shape(B, N, C, G, dtype)) return rc;
    SID_CHECK_ARG(act == SID_ACT_NONE || act == SID_ACT_SILU, "unknown activation %d", act);
    SID_CHECK_ARG(aligned_to_elements((uintptr_t)x | (uintptr_t)y, dtype), "tensors must be aligned to their elements");
    SID_CHECK_ARG(eps >= 0.f, "eps must not be negative");
    const Plan pl = make_plan(B, N, C, G, dtype, (uintptr_t)x | (uintptr_t)y, false);
    if (int rc = check_launch(pl, B, C, G, dtype)) return rc;
    if (plan_bytes(pl) > workspace_bytes) return sid::fail(SID_ENOMEM, "workspace of %zu bytes, %zu needed", workspace_bytes, plan_bytes(pl));
    SID_CHECK_ARG(plan_bytes(pl) == 0 || (workspace && (uintptr_t)workspace % 256 == 0), "workspace must be 256-byte aligned");
    NormParams p = params_of(B, N, C, G, act);
    p.x = (const char*)x; p.out = (char*)y; p.w = weight; p.b = bias; p.mean = mean; p.rstd = rstd; p.eps = eps;
    p.chunks = pl.chunks; p.chunk_rows = pl.chunk_rows; p.out_rows = pl.out_rows;
    p.gc = pl.gc; p.fold = pl.fold;
    p.part = (float2*)workspace;
    p.gpart = (float2*)((char*)workspace + pl.part_bytes);
    return by_dtype(p, pl, dtype, false, (hipStream_t)stream);
}

extern "C" int sid_group_norm_act_bwd(const void* dy, const void* x, const float* weight, const float* bias,
                                      const float* mean, const float* rstd, void* dx, float* dweight, float* dbias,
                                      int B, int N, int C, int G, int act, int dtype,
                                      void* workspace, size_t workspace_bytes, void* stream) {
    SID_CHECK_ARG(dy && x && mean && rstd, "NULL tensor pointer");
    SID_CHECK_ARG(dx || dweight || dbias, "no gradient asked for");
    if (int rc = check_shape(B, N, C, G, dtype)) return rc;
    SID_CHECK_ARG(act == SID_ACT_NONE || act == SID_ACT_SILU, "unknown activation %d", act);
    SID_CHECK_ARG(aligned_to_elements((uintptr_t)x | (uintptr_t)dy | (uintptr_t)dx, dtype), "tensors must be aligned to their elements");
    const Plan pl = make_plan(B, N, C, G, dtype, (uintptr_t)x | (uintptr_t)dy | (uintptr_t)dx, true);
    if (int rc = check_launch(pl, B, C, G, dtype)) return rc;
    if (plan_bytes(pl) > workspace_bytes) return sid::fail(SID_ENOMEM, "workspace of %zu bytes, %zu needed", workspace_bytes, plan_bytes(pl));
    SID_CHECK_ARG(workspace && (uintptr_t)workspace % 256 == 0, "workspace must be 256-byte aligned");
    NormParams p = params_of(B, N, C, G, act);
    p.x = (const char*)x; p.dy = (const char*)dy; p.out = (char*)dx; p.w = weight; p.b = bias;
    p.mean = (float*)mean; p.rstd = (float*)rstd;
    p.chunks = pl.chunks; p.chunk_rows = pl.chunk_rows; p.out_rows = pl.out_rows;
    p.dw = dweight; p.db = dbias;
    char* ws = (char*)workspace;
    p.part = (float2*)ws;
    p.fold = pl.fold;
    p.sums = p.gpart = (float2*)(ws + pl.part_bytes);
    p.chan = pl.chan_bytes && (dweight || dbias) ? (float2*)(ws + pl.part_bytes + pl.sums_bytes) : nullptr;
    return by_dtype(p, pl, dtype, true, (hipStream_t)stream);
}
