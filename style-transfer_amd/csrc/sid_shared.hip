// Shared-prefix attention: decomposition, the joining kernel and the entry points.  Kernels: sid_shared_kernel.hpp.
#include "sid_shared_kernel.hpp"

#include <cmath>

namespace sid_shared {
namespace {

constexpr int kMaxSlots = 128;

// out = sum over slots of 2^(m - M) part / sum of 2^(m - M) l.  A thread owns four columns (quad) of one row and every
// (1 << log_sg)-th slot; 2^log_q quads, so a row has 2^(log_q + log_sg) threads.  They read the row's references and sums
// together, and what they gather from their slots is joined through LDS.
template <typename T>
__global__ void __launch_bounds__(256) combine_kernel(const float* __restrict__ part, const float2* __restrict__ stats, char* __restrict__ out,
                                                      int rows, int d, int slots, int log_q, int log_sg) {
    __shared__ float2 st[16 * kMaxSlots];            // (weight, sum) per row of the workgroup and slot
    __shared__ float4 acc[256];
    __shared__ float tot[256];
    const int tid = threadIdx.x, per_row = 1 << (log_q + log_sg), lr = tid >> (log_q + log_sg);
    const int in_row = tid & (per_row - 1), quad = in_row & ((1 << log_q) - 1), sg = in_row >> log_q;
    const int row = blockIdx.x * (256 / per_row) + lr;
    const bool live = row < rows;
    float2* mine = st + lr * slots;
    for (int s = in_row; s < slots; s += per_row) mine[s] = live ? stats[(long long)s * rows + row] : make_float2(kNegInf, 0.f);
    __syncthreads();
    float top = kNegInf;
    for (int s = 0; s < slots; ++s) top = fmaxf(top, mine[s].x);
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    float total = 0.f;
    if (live && quad * 4 < d) {
        const float* src = part + (long long)row * d + quad * 4;
#pragma unroll 8
        for (int s = sg; s < slots; s += 1 << log_sg) {
            const float2 v = mine[s];
            const float4 o = *(const float4*)(src + (long long)s * rows * d);
            // an empty slot has reference -inf and sum 0; one whose keys gave NaN may have that reference and a NaN sum
            const float w = v.x == kNegInf ? (v.y == 0.f ? 0.f : v.y) : __builtin_amdgcn_exp2f(v.x - top);
            total = __builtin_fmaf(w, v.y, total);
            a.x = __builtin_fmaf(w, o.x, a.x); a.y = __builtin_fmaf(w, o.y, a.y);
            a.z = __builtin_fmaf(w, o.z, a.z); a.w = __builtin_fmaf(w, o.w, a.w);
        }
    }
    for (int h = 1 << log_sg >> 1; h >= 1; h >>= 1) {
        acc[tid] = a;
        tot[tid] = total;
        __syncthreads();
        if (sg < h) {
            const float4 o = acc[tid + (h << log_q)];
            a.x += o.x; a.y += o.y; a.z += o.z; a.w += o.w;
            total += tot[tid + (h << log_q)];
        }
        __syncthreads();
    }
    if (sg == 0 && live && quad * 4 < d) {
        const float inv = total == 0.f ? 0.f : 1.f / total;
        store4<T>(out + ((long long)row * d + quad * 4) * 2, a.x * inv, a.y * inv, a.z * inv, a.w * inv);
    }
}

struct Plan {
    int qt, slots, groups;
    Group g[2];
};

constexpr int kFill = 512;          // workgroups that fill the chip: two on each of 256 CUs

int padded(int items) { return (items + kXcd - 1) / kXcd * kXcd; }
int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

// Splits of a key range of `keys` into at most `fill` workgroups over `items`, each with at least `least` keys.
int splits_for(long long items, long long keys, long long fill, int least) {
    long long s = fill / items;
    if (s > keys / least) s = keys / least;
    return (int)(s < 1 ? 1 : s > kMaxSlots / 2 ? kMaxSlots / 2 : s);
}

// mixed: the parts are held in different formats, so no item may walk both.
Plan make_plan(int B, int Hkv, int G, int n, int d, int P, int S, bool mixed) {
    Plan pl{};
    const long long rows = (long long)n * G;             // of one image
    const int unit = tile_rows(class_of(d));
    pl.qt = 1;
    auto add = [&](int k, int tiles, int rows_of_tile, int splits, int per_image, int by_keys, int segs) {
        pl.g[k] = Group{(int)((long long)Hkv * (per_image ? B : 1) * tiles * splits), tiles, splits, pl.slots, rows_of_tile, per_image, by_keys, segs,
                        Div((unsigned)tiles), Div((unsigned)splits)};
        pl.slots += splits;
        pl.groups = k + 1;
    };
    if (rows > 64) {
        // many rows per image: each tile walks prefix and own keys
        auto items_of = [&](int qt) { return (long long)B * Hkv * ceil_div(rows, 4 * unit * qt); };
        auto splits_of = [&](long long items, long long keys) { return splits_for(items, keys, kFill + items / 2, 512); };
        // 64 rows a wave read every fragment of the keys once for two tiles (d = 40, 4 x 4096 queries: 246 us, 274 with 32), as
        // long as the chip is full all the same (8 x 256 queries on 512 keys, 128 workgroups: 15 us, 10.5 with 32)
        const long long twos = items_of(2);
        pl.qt = two_tiles(class_of(d)) && twos * splits_of(twos, (long long)P + S) >= kFill ? 2 : 1;
        const int tile = 4 * unit * pl.qt, tiles = ceil_div(rows, tile);
        const long long items = items_of(pl.qt);
        if (mixed && P && S) {
            add(0, tiles, tile, splits_of(items, P), 1, 0, 1);
            add(1, tiles, tile, splits_of(items, S), 1, 0, 2);
        } else {
            add(0, tiles, tile, splits_of(items, (long long)P + S), 1, 0, (P ? 1 : 0) | (S ? 2 : 0));
        }
    } else {
        // the chip's workgroups are shared out by the keys that prefix and own parts have to walk
        const long long all = rows * B;
        const int by_keys = all <= unit, ptile = by_keys ? unit : 4 * unit, ptiles = ceil_div(all, ptile), otiles = ceil_div(rows, unit);
        const long long pitems = (long long)Hkv * ptiles, oitems = (long long)B * Hkv * otiles, pwork = pitems * P, owork = oitems * S;
        int k = 0;
        if (P) add(k++, ptiles, ptile, splits_for(pitems, P, kFill * pwork / (pwork + owork) + pitems / 2, by_keys ? 128 : 256), 0, by_keys, 1);
        if (S) add(k++, otiles, unit, splits_for(oitems, S, kFill * owork / (pwork + owork) + oitems / 2, 128), 1, 1, 2);
        if (!k) add(0, otiles, unit, 1, 1, 1, 0);        // no keys at all: zeros
    }
    return pl;
}

int check_shape(int B, int Hq, int Hkv, int n, int d, int P, int S) {
    SID_CHECK_ARG(B >= 1 && Hq >= 1 && Hkv >= 1 && n >= 1, "B, heads and queries must be >= 1");
    SID_CHECK_ARG(P >= 0 && S >= 0, "key counts must not be negative");
    SID_CHECK_ARG(Hq % Hkv == 0, "%d query heads do not divide among %d key/value heads", Hq, Hkv);
    SID_CHECK_ARG(d >= 8 && d <= 256 && d % 8 == 0, "head_dim must be a multiple of 8 in [8, 256], got %d", d);
    SID_CHECK_ARG((long long)B * n * Hq < (1 << 24) && P < (1 << 30) && S < (1 << 30), "too many rows or keys");
    return SID_OK;
}

size_t plan_bytes(const Plan& pl, long long rows, int d) {
    return pl.slots <= 1 ? 0 : sid::align_up((size_t)pl.slots * rows * d * 4, 256) + (size_t)pl.slots * rows * sizeof(float2);
}

int check_source(const sid_kv_source* s, int keys, int d, const char* what) {
    SID_CHECK_ARG(s && s->k && s->v, "%s: NULL pointer", what);
    SID_CHECK_ARG(s->fmt == SID_KV_NONE || s->fmt == SID_KV_INT8 || s->fmt == SID_KV_E4M3, "%s: unknown format %d", what, s->fmt);
    const int es = s->fmt == SID_KV_NONE ? 2 : 1, unit = s->fmt == SID_KV_NONE ? 16 : 8;
    const long long st[6] = {s->k_stride[0], s->k_stride[1], s->k_stride[2], s->v_stride[0], s->v_stride[1], s->v_stride[2]};
    SID_CHECK_ARG((uintptr_t)s->k % unit == 0 && (uintptr_t)s->v % unit == 0, "%s: keys and values must be %d-byte aligned", what, unit);
    for (long long x : st) SID_CHECK_ARG(x * es % unit == 0, "%s: rows must be %d-byte aligned", what, unit);
    for (int i = 2; i < 6; i += 3)
        SID_CHECK_ARG(st[i] >= 0 && st[i] * es < (1 << 24), "%s: distance between tokens out of range", what);
    SID_CHECK_ARG(s->fmt == SID_KV_NONE || d >= 16, "%s: 8-bit rows need a head_dim of 16 or more", what);
    if (s->fmt != SID_KV_NONE) SID_CHECK_ARG(s->k_scale && s->v_scale, "%s: scales missing", what);
    return SID_OK;
}

void fill_source(Source& o, const sid_kv_source* s) {
    const int es = s->fmt == SID_KV_NONE ? 2 : 1;
    o.k = (const char*)s->k; o.v = (const char*)s->v;
    o.ks = s->k_scale; o.vs = s->v_scale;
    o.kb = s->k_stride[0] * es; o.kh = s->k_stride[1] * es; o.kn = (int)(s->k_stride[2] * es);
    o.vb = s->v_stride[0] * es; o.vh = s->v_stride[1] * es; o.vn = (int)(s->v_stride[2] * es);
    o.sb = s->scale_stride[0]; o.sh = s->scale_stride[1];
}

}  // namespace
}  // namespace sid_shared

using namespace sid_shared;

extern "C" size_t sid_shared_attn_workspace_bytes(int B, int Hq, int Hkv, int n, int d, int P, int S, int mixed) {
    if (check_shape(B, Hq, Hkv, n, d, P, S)) return 0;
    const size_t need = plan_bytes(make_plan(B, Hkv, Hq / Hkv, n, d, P, S, mixed != 0), (long long)B * n * Hq, d);
    return need ? need : 256;
}

extern "C" int sid_shared_attn_fwd(const void* q, const long long* q_stride, const sid_kv_source* prefix, const sid_kv_source* own,
                                   const int* own_len, void* out, int B, int Hq, int Hkv, int n, int d, int P, int S,
                                   float scale, int causal, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
    SID_CHECK_ARG(q && q_stride && out, "NULL pointer");
    if (int rc = check_shape(B, Hq, Hkv, n, d, P, S)) return rc;
    SID_CHECK_ARG(dtype == SID_DTYPE_BF16 || dtype == SID_DTYPE_F16, "queries must be bf16 or f16, got dtype %d", dtype);
    SID_CHECK_ARG(scale > 0.f && std::isfinite(scale), "scale must be positive and finite");
    SID_CHECK_ARG((uintptr_t)q % 16 == 0 && (uintptr_t)out % 8 == 0, "queries must be 16-byte aligned, the output 8-byte");
    for (int i = 0; i < 3; ++i) SID_CHECK_ARG(q_stride[i] % 8 == 0, "query rows must be 16-byte aligned");
    if (P) if (int rc = check_source(prefix, P, d, "prefix")) return rc;
    if (S) if (int rc = check_source(own, S, d, "own part")) return rc;

    const int fmt[2] = {P ? prefix->fmt : SID_KV_NONE, S ? own->fmt : SID_KV_NONE};
    const Plan pl = make_plan(B, Hkv, Hq / Hkv, n, d, P, S, P && S && fmt[0] != fmt[1]);
    long long workgroups = 0;
    for (int g = 0; g < pl.groups; ++g) workgroups += padded(pl.g[g].items);
    SID_CHECK_ARG(workgroups < (1 << 24), "too many rows");                       // a launch holds fewer than 2^32 threads in x
    const long long rows = (long long)B * n * Hq;
    const size_t need = plan_bytes(pl, rows, d);
    if (need > workspace_bytes) return sid::fail(SID_ENOMEM, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
    SID_CHECK_ARG(need == 0 || (workspace && (uintptr_t)workspace % 256 == 0), "workspace must be 256-byte aligned");
    Params p{};
    p.q = (const char*)q;
    p.qb = q_stride[0] * 2; p.qh = q_stride[1] * 2; p.qn = q_stride[2] * 2;
    if (P) fill_source(p.src[0], prefix);
    if (S) fill_source(p.src[1], own);
    p.own_len = own_len;
    p.out = (char*)out;
    if (need) {
        p.part = (float*)workspace;
        p.stats = (float2*)((char*)workspace + sid::align_up((size_t)pl.slots * rows * d * 4, 256));
    }
    p.B = B; p.Hq = Hq; p.Hkv = Hkv; p.G = Hq / Hkv; p.n = n; p.d = d; p.P = P; p.S = S; p.causal = causal != 0;
    p.c = scale * 1.4426950408889634f;
    p.by_B = Div((unsigned)B); p.by_G = Div((unsigned)p.G); p.by_n = Div((unsigned)n);
    const hipStream_t st = (hipStream_t)stream;
    // one launch for the groups whose parts are held alike
    for (int g = 0; g < pl.groups;) {
        const int f = fmt[pl.g[g].segs == 2];
        const bool both = g + 1 < pl.groups && fmt[pl.g[g + 1].segs == 2] == f;
        p.g[0] = pl.g[g];
        p.g[1] = both ? pl.g[g + 1] : Group{};
        p.blocks0 = padded(p.g[0].items);
        const unsigned grid = (unsigned)(p.blocks0 + padded(p.g[1].items));
        int rc;
        if (dtype == SID_DTYPE_BF16) rc = f != SID_KV_NONE ? launch_bf16_codes(p, f, pl.qt, grid, st) : launch_bf16(p, pl.qt, grid, st);
        else rc = f != SID_KV_NONE ? launch_f16_codes(p, f, pl.qt, grid, st) : launch_f16(p, pl.qt, grid, st);
        if (rc) return rc;
        g += both ? 2 : 1;
    }
    if (need) {
        // quads of a row to a power of two; slots shared by up to 16 threads (d <= 64; 8 to 128, 4 above) while that leaves
        // each one a few
        int log_q = 4, log_sg = 0;
        while ((4 << log_q) < d) ++log_q;
        while (log_sg < 8 - log_q && (4 << log_sg) < pl.slots) ++log_sg;
        const int per_block = 256 >> (log_q + log_sg);
        const unsigned grid = (unsigned)((rows + per_block - 1) / per_block);
        if (dtype == SID_DTYPE_BF16) hipLaunchKernelGGL(combine_kernel<__bf16>, dim3(grid), dim3(256), 0, st, p.part, p.stats, p.out, (int)rows, d, pl.slots, log_q, log_sg);
        else hipLaunchKernelGGL(combine_kernel<_Float16>, dim3(grid), dim3(256), 0, st, p.part, p.stats, p.out, (int)rows, d, pl.slots, log_q, log_sg);
        SID_CHECK_HIP(hipGetLastError());
    }
    return SID_OK;
}
