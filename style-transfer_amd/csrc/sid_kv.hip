// Key/value cache in 8 bits: quantised as it is written, read back as numbers.
//
// A cache holds codes (B, H, S, d), 8 bits each (int8 or e4m3), and one f32 scale per row (B, H, S); the number a code
// stands for is code * scale.  A row is written with the scale that maps its largest magnitude to the largest code:
//   scale = amax / top,  code = round_to_nearest_even(x * (top / amax)),  top = 127 (int8) or 448 (e4m3)
// in f32 (the quotient is formed once per row, so a value within an f32 rounding of the middle between two codes may
// go to either).  A row whose amax is below 2^-100 is stored as zeros with scale 0; a row that holds an infinity or a
// NaN gets the scale NaN and zero codes and reads back as NaN.
//
// Writing reads d elements and writes d + 4 bytes per row, reading the reverse: both are bound by memory.  A write works
// on groups of lanes of 8 elements per lane (one 16-byte load of 16-bit values, one 8-byte store of codes), heads
// fastest, so a workgroup reads whole token rows and writes runs of consecutive tokens of each head.  A read is one
// flat copy per (image, head), since rows follow each other on both sides.
// Measured: writing 4 x 4096 tokens of 8 x 40 f32 (53 MB) 13.0 us, 4.1 TB/s; reading 8 x 4001 tokens of 8 x 80 as f16
// (125 MB) 20.5 us, 6.1 TB/s (a 1 GiB copy on the same card: 5.1 TB/s); one token of 16 sequences 3.7 us.
#include "sid_common.h"

#include <cstdint>

namespace {

constexpr float kTiny = 7.8886090522101181e-31f;       // 2^-100

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;

template <int DT>
__device__ __forceinline__ void load8(const char* p, float* f) {
    if constexpr (DT == SID_DTYPE_F32) {
        const float4 a = ((const float4*)p)[0], b = ((const float4*)p)[1];
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    } else if constexpr (DT == SID_DTYPE_BF16) {
        const bf16x8 v = *(const bf16x8*)p;
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = (float)v[e];
    } else {
        const f16x8 v = *(const f16x8*)p;
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = (float)v[e];
    }
}

template <int DT>
__device__ __forceinline__ void store8(char* p, const float* f) {
    if constexpr (DT == SID_DTYPE_F32) {
        ((float4*)p)[0] = make_float4(f[0], f[1], f[2], f[3]);
        ((float4*)p)[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else if constexpr (DT == SID_DTYPE_BF16) {
        bf16x8 v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (__bf16)f[e];
        *(bf16x8*)p = v;
    } else {
        f16x8 v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (_Float16)f[e];
        *(f16x8*)p = v;
    }
}

struct WriteParams {
    const char* src[2];             // keys, values
    long long sb[2], sh[2], sn[2];  // their strides over images, heads and tokens, in bytes
    uint8_t* codes[2];
    float* scale[2];
    const int *start, *length;
    long long rows;                 // B * n * H
    int H, n, S, d, lanes_log2;
};

template <int DT, int FMT>
__global__ void __launch_bounds__(256) kv_write(WriteParams p) {
    const int lanes = 1 << p.lanes_log2, lane = threadIdx.x & (lanes - 1);
    const int per_block = 256 >> p.lanes_log2;
    const long long r = (long long)blockIdx.x * per_block + (threadIdx.x >> p.lanes_log2);
    if (r >= p.rows) return;                             // whole groups leave: the exchanges below stay inside a group
    const int h = (int)(r % p.H);
    const long long tok = r / p.H;
    const int i = (int)(tok % p.n), b = (int)(tok / p.n);
    const long long at = (long long)p.start[b] + i;
    if (at < 0 || at >= p.S || (p.length && i >= p.length[b])) return;
    const bool live = lane * 8 < p.d;
    float f[2][8];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[x][e] = 0.f;
        if (live) load8<DT>(p.src[x] + b * p.sb[x] + h * p.sh[x] + i * p.sn[x] + (long long)lane * 8 * (DT == SID_DTYPE_F32 ? 4 : 2), f[x]);
    }
    const long long row = ((long long)b * p.H + h) * p.S + at;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        // magnitudes compare as integers, infinities and NaN above all numbers
        uint32_t m = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(f[x][e]) & 0x7fffffffu);
        for (int off = 1; off < lanes; off <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, off));
        const float amax = __uint_as_float(m), top = FMT == SID_KV_INT8 ? 127.f : 448.f;
        const bool bad = m >= 0x7f800000u, some = !bad && amax >= kTiny;
        const float inv = some ? top / amax : 0.f;
        uint32_t w[2] = {0u, 0u};
#pragma unroll
        for (int e = 0; e < 8; ++e) f[x][e] = bad ? 0.f : fminf(fmaxf(f[x][e] * inv, -top), top);
        if constexpr (FMT == SID_KV_INT8) {
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e / 4] |= ((uint32_t)(int)rintf(f[x][e]) & 255u) << (8 * (e & 3));
        } else {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                int v = __builtin_amdgcn_cvt_pk_fp8_f32(f[x][4 * e], f[x][4 * e + 1], 0, false);
                w[e] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[x][4 * e + 2], f[x][4 * e + 3], v, true);
            }
        }
        if (live) *(uint2*)(p.codes[x] + row * p.d + lane * 8) = make_uint2(w[0], w[1]);
        if (lane == 0) p.scale[x][row] = bad ? __builtin_nanf("") : some ? amax / top : 0.f;
    }
}

struct ReadParams {
    const uint8_t* codes[2];
    const float* scale[2];
    char* out[2];                   // (B, H, n, d)
    const int* start;
    int H, n, S, d, d8;             // d8 = d / 8
    unsigned chunks;                // n * d8, of 8 elements
    unsigned long long inv_d8;      // ceil(2^32 / d8): chunk / d8 = chunk * inv >> 32 while chunk * d8 < 2^32
};

template <int DT, int FMT>
__global__ void __launch_bounds__(256) kv_read(ReadParams p) {
    const int bh = blockIdx.y, b = bh / p.H;
    const long long start = p.start[b];
    constexpr int R = 4;
    uint2 code[2][R];
    float scale[2][R];
    const unsigned c0 = blockIdx.x * (256u * R) + threadIdx.x;
#pragma unroll
    for (int k = 0; k < R; ++k) {
        const unsigned c = c0 + k * 256u;
        const unsigned i = (unsigned)((c * p.inv_d8) >> 32);
        const long long at = start + i;
        const bool in = c < p.chunks && at >= 0 && at < p.S;
        const long long row = (long long)bh * p.S + at;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            code[x][k] = make_uint2(0u, 0u);
            scale[x][k] = 0.f;
            if (in) {
                code[x][k] = *(const uint2*)(p.codes[x] + row * p.d + (size_t)(c - i * (unsigned)p.d8) * 8);
                scale[x][k] = p.scale[x][row];
            }
        }
    }
#pragma unroll
    for (int k = 0; k < R; ++k) {
        const unsigned c = c0 + k * 256u;
        if (c >= p.chunks) break;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            float f[8];
            const uint32_t w[2] = {code[x][k].x, code[x][k].y};
            if constexpr (FMT == SID_KV_INT8) {
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = (float)(int8_t)(w[e / 4] >> (8 * (e & 3)));
            } else {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[e], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[e], true);
                    f[4 * e] = lo[0]; f[4 * e + 1] = lo[1]; f[4 * e + 2] = hi[0]; f[4 * e + 3] = hi[1];
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] *= scale[x][k];
            store8<DT>(p.out[x] + ((size_t)bh * p.chunks + c) * (8 * (DT == SID_DTYPE_F32 ? 4 : 2)), f);
        }
    }
}

int check_cache(int B, int H, int S, int d, int fmt) {
    SID_CHECK_ARG(B >= 1 && H >= 1 && S >= 1, "B, H, S must be >= 1");
    SID_CHECK_ARG(d >= 8 && d <= 256 && d % 8 == 0, "head_dim must be a multiple of 8 in [8, 256], got %d", d);
    SID_CHECK_ARG(fmt == SID_KV_INT8 || fmt == SID_KV_E4M3, "unknown cache format %d", fmt);
    SID_CHECK_ARG((long long)B * H < (1 << 16), "too many (image, head) pairs");
    return SID_OK;
}

template <int DT>
int launch_write(const WriteParams& p, int fmt, unsigned grid, hipStream_t st) {
    if (fmt == SID_KV_INT8) hipLaunchKernelGGL((kv_write<DT, SID_KV_INT8>), dim3(grid), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((kv_write<DT, SID_KV_E4M3>), dim3(grid), dim3(256), 0, st, p);
    SID_CHECK_HIP(hipGetLastError());
    return SID_OK;
}

template <int DT>
int launch_read(const ReadParams& p, int fmt, dim3 grid, hipStream_t st) {
    if (fmt == SID_KV_INT8) hipLaunchKernelGGL((kv_read<DT, SID_KV_INT8>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((kv_read<DT, SID_KV_E4M3>), grid, dim3(256), 0, st, p);
    SID_CHECK_HIP(hipGetLastError());
    return SID_OK;
}

}  // namespace

extern "C" int sid_kv_cache_write(const void* k, const void* v, const long long* k_strides, const long long* v_strides,
                                  void* k_codes, void* v_codes, float* k_scale, float* v_scale,
                                  const int* start, const int* length,
                                  int B, int H, int n, int S, int d, int dtype, int fmt, void* stream) {
    SID_CHECK_ARG(k_strides && v_strides && k_codes && v_codes && k_scale && v_scale && start, "NULL pointer");
    if (int rc = check_cache(B, H, S, d, fmt)) return rc;
    SID_CHECK_ARG(n >= 0, "n must not be negative");
    SID_CHECK_ARG(dtype == SID_DTYPE_F32 || dtype == SID_DTYPE_BF16 || dtype == SID_DTYPE_F16, "unknown dtype %d", dtype);
    if (n == 0) return SID_OK;
    SID_CHECK_ARG(k && v, "NULL pointer");
    const int es = dtype == SID_DTYPE_F32 ? 4 : 2;
    WriteParams p{};
    const void* src[2] = {k, v};
    const long long* strides[2] = {k_strides, v_strides};
    for (int x = 0; x < 2; ++x) {
        SID_CHECK_ARG((uintptr_t)src[x] % 16 == 0, "keys and values must be 16-byte aligned");
        for (int a = 0; a < 3; ++a) SID_CHECK_ARG(strides[x][a] * es % 16 == 0, "rows of keys and values must be 16-byte aligned");
        p.src[x] = (const char*)src[x];
        p.sb[x] = strides[x][0] * es; p.sh[x] = strides[x][1] * es; p.sn[x] = strides[x][2] * es;
    }
    SID_CHECK_ARG((uintptr_t)k_codes % 8 == 0 && (uintptr_t)v_codes % 8 == 0, "codes must be 8-byte aligned");
    p.codes[0] = (uint8_t*)k_codes; p.codes[1] = (uint8_t*)v_codes;
    p.scale[0] = k_scale; p.scale[1] = v_scale;
    p.start = start; p.length = length;
    p.rows = (long long)B * n * H;
    p.H = H; p.n = n; p.S = S; p.d = d;
    while ((8 << p.lanes_log2) < d) ++p.lanes_log2;
    const long long per_block = 256 >> p.lanes_log2, grid = (p.rows + per_block - 1) / per_block;
    SID_CHECK_ARG(grid < (1LL << 24), "too many rows");            // a launch holds fewer than 2^32 threads in x
    if (dtype == SID_DTYPE_F32) return launch_write<SID_DTYPE_F32>(p, fmt, (unsigned)grid, (hipStream_t)stream);
    if (dtype == SID_DTYPE_BF16) return launch_write<SID_DTYPE_BF16>(p, fmt, (unsigned)grid, (hipStream_t)stream);
    return launch_write<SID_DTYPE_F16>(p, fmt, (unsigned)grid, (hipStream_t)stream);
}

extern "C" int sid_kv_cache_read(const void* k_codes, const void* v_codes, const float* k_scale, const float* v_scale,
                                 void* k, void* v, const int* start,
                                 int B, int H, int n, int S, int d, int dtype, int fmt, void* stream) {
    SID_CHECK_ARG(k_codes && v_codes && k_scale && v_scale && start, "NULL pointer");
    if (int rc = check_cache(B, H, S, d, fmt)) return rc;
    SID_CHECK_ARG(n >= 0, "n must not be negative");
    SID_CHECK_ARG(dtype == SID_DTYPE_F32 || dtype == SID_DTYPE_BF16 || dtype == SID_DTYPE_F16, "unknown dtype %d", dtype);
    if (n == 0) return SID_OK;
    SID_CHECK_ARG(k && v, "NULL pointer");
    SID_CHECK_ARG((uintptr_t)k_codes % 8 == 0 && (uintptr_t)v_codes % 8 == 0, "codes must be 8-byte aligned");
    SID_CHECK_ARG((uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0, "keys and values must be 16-byte aligned");
    // chunk / d8 by a multiplication: right while chunk * d8 < 2^32 (the launch rounds chunks up by at most 1023)
    SID_CHECK_ARG(((long long)n * (d / 8) + 1024) * (d / 8) < (1LL << 32), "n too large");
    ReadParams p{};
    p.codes[0] = (const uint8_t*)k_codes; p.codes[1] = (const uint8_t*)v_codes;
    p.scale[0] = k_scale; p.scale[1] = v_scale;
    p.out[0] = (char*)k; p.out[1] = (char*)v;
    p.start = start;
    p.H = H; p.n = n; p.S = S; p.d = d; p.d8 = d / 8;
    p.chunks = (unsigned)n * (unsigned)p.d8;
    p.inv_d8 = ((1ull << 32) + p.d8 - 1) / p.d8;
    const dim3 grid((p.chunks + 1023) / 1024, (unsigned)(B * H));
    if (dtype == SID_DTYPE_F32) return launch_read<SID_DTYPE_F32>(p, fmt, grid, (hipStream_t)stream);
    if (dtype == SID_DTYPE_BF16) return launch_read<SID_DTYPE_BF16>(p, fmt, grid, (hipStream_t)stream);
    return launch_read<SID_DTYPE_F16>(p, fmt, grid, (hipStream_t)stream);
}
