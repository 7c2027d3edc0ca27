// Attention of a batch whose sequences share a prefix of keys and values: device code and launch templates.
//
// Row r = (b n + i) G + g of key/value head h is query i of head h G + g of image b.  It attends to the P keys of the
// prefix (one copy for the whole batch) and to the first lim(r) of its image's own S keys under one softmax:
//   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  s_j = scale q.k_j,
// lim = own_len[b], or with the causal order min(own_len, max(0, own_len - n + 1 + i)).  A row without keys gives zeros.
//
// Work items.  An item is a tile of rows times a range of key tiles; it yields the un-normalised output, the softmax
// reference and the row sum, which combine_kernel joins when a row has more than one.
//   Many rows per image: items are row tiles of one image and walk the prefix, then the own keys.
//   Few rows per image (decoding): the rows of ALL images that share a key/value head stand in the same tiles against the
//   prefix, so the prefix is read once for the batch and not once per image; the own keys are items of their own.
//   Long key ranges are split over items until the chip is full.
//
// Two ways for a workgroup of four waves to share an item:
//   rows   each wave owns 32 QT rows, key tiles of 64 are staged for all four (double-buffered, one barrier a tile);
//   keys   up to 32 rows: every wave takes every fourth tile of 32 keys through its own buffer, without barriers, and
//          the four results are joined at the end.  One row (a single token) costs the matrix unit as much as 32, which
//          is still below the time that the keys take to arrive.
//
// MFMA 32x32x16, keys on rows and queries on lanes as in sid_attn_kernel.hpp: S^T = K Q^T, whose accumulator rounded to
// 16 bits is the B operand of O^T += V^T P^T when the key order of the A operand follows the accumulator's.  V stays
// row-major in LDS; ds_read_b64_tr_b16 hands every lane four consecutive keys of its column.  Where head_dim leaves a
// spare column in V's last block of 32, that column holds ones and the product also yields the row sum.
// Heads wider than 128 take 16x16x32 and 16 rows a wave (Rows16): 32 rows of them do not fit 256 registers.
// Tiles go through registers to LDS: the next tile's loads are in flight while this one is computed, and keys behind the
// end become zeros.  8-bit codes become the call's 16-bit type on the way: key codes as they are (both types hold them
// exactly; their scale multiplies the f32 logits, because a rounding of the keys would shift a logit by 2^-9 of the sum of
// |q k|, twice the error of everything else at |logit| = 5), value codes times their scale, rounded once.
//
// Measured: 4 images of 4096 queries, 8 heads of 40, 4096 + 4096 keys 233 us, 740 TFLOP/s (a tile of 64 keys takes a SIMD
// about 1930 cycles, which is its products' 900 and its vector work's 1050 one after the other; d = 128 565 us, 970 TFLOP/s);
// one token of 32 sequences, 32 / 8 heads of 128, 32768 + 1024 keys 49 us + 6 us to join, 4.2 TB/s (bound by memory; on
// int8 codes 49 us for both); five tokens of 16 sequences on int8 codes, 16 / 4 heads of 128, 8191 + 333 keys 28 us + 5 us
// (21 MB of partial results written and read, and every code converted for three row tiles); one token of 4 sequences on
// 1023 + 128 keys 6.4 us + 3.4 us (a workgroup's chain of loads, products and join).  Heads of 160 and 256, 4 images of 2048
// queries on 2048 + 2048 keys: 440 and 629 us, 390 and 437 TFLOP/s (Rows16 reads each K fragment right before its product,
// for 16 rows only).
#pragma once
#include "sid_common.h"

#include <cstdint>
#include <type_traits>

namespace sid_shared {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;     // a native vector: stays in registers
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;

constexpr int kXcd = 8;
constexpr float kNegInf = -__builtin_huge_valf();
constexpr int kVector = 0x2 | 0x4 | 0x400;   // sched_barrier: vector, scalar and transcendental instructions may pass
constexpr float kNone = -3e38f;       // softmax reference before the first key: finite, so that no difference is NaN

struct Source {                      // keys and values of the prefix, or of the images' own part
    const char *k, *v;
    const float *ks, *vs;            // 8-bit formats: one scale per row
    long long kb, kh, vb, vh;        // bytes from image to image, head to head
    long long sb, sh;                // the same for the scales, in floats
    int kn, vn;                      // bytes from key to key
};

struct Div {                         // division by a host constant: n / d for 0 <= n < 2^31
    unsigned mul, shift;
    Div() = default;
    explicit Div(unsigned d) : mul(0), shift(0) {
        while ((1ull << shift) < d) ++shift;
        mul = (unsigned)((((1ull << shift) - d) << 32) / d + 1);
    }
    __device__ __forceinline__ int operator()(int n) const { return (int)((__umulhi(mul, (unsigned)n) + (unsigned)n) >> shift); }
};

struct Group {                       // work items of one kind
    int items, tiles, splits, slot0, tile_rows;
    int per_image;                   // row tiles of one image, or of all images together
    int keys_way;                    // waves share the keys (up to 32 rows) instead of the rows
    int segs;                        // 1: prefix, 2: own, 3: both
    Div by_tiles, by_splits;
};

struct Params {
    const char* q;
    long long qb, qh, qn;            // strides in bytes
    Source src[2];                   // prefix, own
    const int* own_len;
    char* out;                       // (B, n, Hq, d)
    float* part;                     // [slot][B n Hq][d], or null: one item per row, which writes `out`
    float2* stats;                   // [slot][B n Hq]: softmax reference (log2 domain), row sum; 0 = nothing in it
    int B, Hq, Hkv, G, n, d, P, S, causal;
    float c;                         // scale * log2(e)
    int blocks0;                     // workgroups of group 0 (a multiple of 8)
    Group g[2];
    Div by_B, by_G, by_n;
};

template <typename T> struct Ops;
template <> struct Ops<__bf16> {
    using V8 = bf16x8;
    static constexpr uint16_t kExp = 0x7f80, kOne = 0x3f80;
    static constexpr float kBias = 0.f;
    static __device__ __forceinline__ f32x16 mfma(V8 a, V8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ f32x4 mfma(V8 a, V8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Ops<_Float16> {
    using V8 = f16x8;
    static constexpr uint16_t kExp = 0x7c00, kOne = 0x3c00;
    // probabilities reach 2^(8 + 6), inside half's range; the smallest it can tell from zero is 2^-30 of the largest
    static constexpr float kBias = 6.f;
    static __device__ __forceinline__ f32x16 mfma(V8 a, V8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ f32x4 mfma(V8 a, V8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

// x of the lane's own half and of lane ^ 32: (lower half's, upper half's) in every lane
__device__ __forceinline__ float2 both_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// (even row's, odd row's) of the lane's pair of 16-lane rows, in every lane
__device__ __forceinline__ float2 both_rows(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// The head-dim classes: KS steps of 16 in q.k, DVB blocks of 32 in V, LPR lanes that stage one row (8 elements each).
template <int KS> struct Dims {
    static constexpr int DVB = (KS + 1) / 2;
    static constexpr int LPR = KS <= 4 ? 8 : KS <= 8 ? 16 : 32;
    static constexpr int KSTR = KS * 16 + 8, VSTR = DVB * 32 + 8;        // LDS row strides in elements (pads spread banks)
    // 128 rows: 2 x 64 (rows way) = 4 x 32 (keys way)
    static constexpr int KELEMS = 128 * KSTR, VELEMS = 128 * VSTR;
    static constexpr int MSTR = DVB * 32 + 4;                            // joining four waves: [4][32][MSTR] floats
    static constexpr size_t kStage = (size_t)(KELEMS + VELEMS) * 2;
    static constexpr size_t kJoin = (size_t)(4 * 32 * MSTR + 2 * 4 * 32) * 4;
    static constexpr size_t kRowData = kStage > kJoin ? kStage : kJoin;              // then per key row a scale and a flag
    static constexpr size_t kLds = kRowData + 128 * 8;
    static constexpr bool kWide = KS > 8;
    static constexpr int ROWS = kWide ? 16 : 32;     // rows of one MFMA tile
    static constexpr int NS = kWide ? 1 : 2;         // sub-tiles of 32 keys whose logits are in registers together
};

// Keys and values of one (image, head) of a part, as a loop over its tiles reads them.
struct Stream {
    const char *k, *v;
    const float *ks, *vs;
    int kn, vn, end;                 // keys from `end` on are not there

    __device__ __forceinline__ Stream(const Params& p, int seg, int b, int h, int keys) {
        const Source& s = p.src[seg];
        const int bi = seg ? b : 0;
        k = s.k + bi * s.kb + h * s.kh;
        v = s.v + bi * s.vb + h * s.vh;
        ks = s.ks + bi * s.sb + h * s.sh;
        vs = s.vs + bi * s.sb + h * s.sh;
        kn = s.kn; vn = s.vn; end = keys;
    }
};

// One key tile on its way from memory to LDS.  NT threads, KT keys.
// Loads are issued on one path, without a condition or a cleared register among them (rows behind the end read the last
// one): a write to a register that an earlier load may still fill waits for that load, and so for the whole latency, and
// where two paths meet the compiler copies what one of them loaded, which waits as well.  store_v()
// clears what was not there; the logits of such keys are masked.
template <typename T, int KS, int NT, int KT, int FMT>
struct Stager {
    using D = Dims<KS>;
    static constexpr bool CODES = FMT != SID_KV_NONE;
    // 16 bytes of every RPP-th row.  Codes: a lane takes 16 of them (half as many lanes a row, half as many loads), the last
    // one of a row those that end it, so rows of 8 (mod 16) codes overlap there and nothing is read behind a row.
    static constexpr int LANES = CODES ? D::LPR / 2 : D::LPR, RPP = NT / LANES, NJ = KT / RPP, NC = CODES ? NJ : 1;
    // a tile waits in registers while the one before it is computed, unless that would take more than 64 of them
    static constexpr bool kAhead = NJ <= 8;
    u32x4 k[NJ], v[NJ];
    float ks[NC], vs[NC];
    int left;                        // rows of the tile that are there, KT at most

    static __device__ __forceinline__ int col_of(const Params& p, int t) {
        return CODES ? min(t % LANES * 16, p.d - 16) : min(t % LANES * 8, p.d - 8);      // lanes behind head_dim repeat its end
    }
    __device__ __forceinline__ void load_k(const Params& p, const Stream& s, int key0, int t) {
        left = min(KT, s.end - key0);
        load_one(p, s.k + (long long)key0 * s.kn, s.ks + key0, s.kn, t, k, ks);
    }
    __device__ __forceinline__ void load_v(const Params& p, const Stream& s, int key0, int t) {
        load_one(p, s.v + (long long)key0 * s.vn, s.vs + key0, s.vn, t, v, vs);
    }
    __device__ __forceinline__ void load(const Params& p, const Stream& s, int key0, int t) {
        load_k(p, s, key0, t);
        load_v(p, s, key0, t);
    }
    __device__ __forceinline__ void load_one(const Params& p, const char* from, const float* scales, int pitch, int t, u32x4 (&to)[NJ],
                                             float (&sc)[NC]) const {
        const int row = t / LANES, col = col_of(p, t) * (CODES ? 1 : 2);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const unsigned r = min(row + j * RPP, left - 1);
            to[j] = *(const u32x4*)(from + (__umul24(r, (unsigned)pitch) + (unsigned)col));        // pitch < 2^24
            if (CODES) sc[j % NC] = scales[r];
        }
    }

    // eight codes as numbers of type T, times `scale`
    static __device__ __forceinline__ u32x4 numbers(uint32_t w0, uint32_t w1, float scale) {
        float f[8];
        // the words as they are from here on: seen through, the compiler would hold every byte in a register of its own from
        // the load on (389 registers)
        asm("" : "+v"(w0), "+v"(w1));
        const uint32_t w[2] = {w0, w1};
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
        typename Ops<T>::V8 o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = (T)(f[e] * scale);
        return __builtin_bit_cast(u32x4, o);
    }

    __device__ __forceinline__ void store_k(const Params& p, T* kl, float* scale, int t) {
        const int row = t / LANES, col = col_of(p, t);
        if (!CODES && t % LANES * 8 >= p.d) return;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            T* to = kl + (row + j * RPP) * D::KSTR + col;
            if (CODES) {
                *(u32x4*)to = numbers(k[j].x, k[j].y, 1.f);
                *(u32x4*)(to + 8) = numbers(k[j].z, k[j].w, 1.f);
                if (t % LANES == 0) scale[row + j * RPP] = ks[j % NC] * p.c;
            } else {
                *(u32x4*)to = k[j];
            }
        }
    }

    // `edge`: keys that some rows of the tile do not see are in it.  Their probability is zero, but zero times an
    // infinity or a NaN is not: such values become zeros and the key is flagged (rows that do see it turn NaN).
    __device__ __forceinline__ void store_v(const Params& p, T* vl, bool edge, int* bad, int t) {
        const int row = t / LANES, col = col_of(p, t);
        if (!CODES && t % LANES * 8 >= p.d) return;
        // all but a part's last tiles need neither test of put_v (heads of 160: 468 -> 431 us)
        if (!edge && left >= KT) {
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                T* to = vl + (row + j * RPP) * D::VSTR + col;
                if (CODES) {
                    *(u32x4*)to = numbers(v[j].x, v[j].y, vs[j % NC]);
                    *(u32x4*)(to + 8) = numbers(v[j].z, v[j].w, vs[j % NC]);
                } else {
                    *(u32x4*)to = v[j];
                }
            }
            return;
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            if (CODES) {
                put_v(vl, row + j * RPP, col, numbers(v[j].x, v[j].y, vs[j % NC]), edge, bad);
                put_v(vl, row + j * RPP, col + 8, numbers(v[j].z, v[j].w, vs[j % NC]), edge, bad);
            } else {
                put_v(vl, row + j * RPP, col, v[j], edge, bad);
            }
        }
    }

    __device__ __forceinline__ void put_v(T* vl, int r, int col, u32x4 c, bool edge, int* bad) const {
        if (left < KT && r >= left) c = u32x4{0u, 0u, 0u, 0u};
        if (edge) {
            uint32_t w[4] = {c.x, c.y, c.z, c.w};
            bool any = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t E = Ops<T>::kExp;
                if ((w[e] & E) == E) { w[e] &= 0xffff0000u; any = true; }
                if ((w[e] & (E << 16)) == (E << 16)) { w[e] &= 0xffffu; any = true; }
            }
            c = u32x4{w[0], w[1], w[2], w[3]};
            if (any) bad[r] = 1;
        }
        *(u32x4*)(vl + r * D::VSTR + col) = c;
    }
};

// Query row r of key/value head h: its place in memory and its number in the sequence
__device__ __forceinline__ int query_of(const Params& p, int h, int r, const char*& src) {
    const int tok = p.by_G(r), g = r - tok * p.G, b = p.by_n(tok), i = tok - b * p.n;
    src = p.q + b * p.qb + (long long)(h * p.G + g) * p.qh + i * p.qn;
    return i;
}

// Softmax state of QT tiles of 32 queries (one query per lane pair) and their output accumulators.
template <typename T, int KS, int QT, bool ONES>
struct Rows32 {
    using D = Dims<KS>;
    using V8 = typename Ops<T>::V8;
    V8 q[QT][KS];
    f32x16 o[QT][D::DVB];
    float m[QT], l[QT];              // softmax reference (log2 domain); row sum of this lane's keys (unless ONES)
    int lim[QT];                     // own keys that the row sees

    __device__ __forceinline__ void init(const Params& p, int h, int row_begin, int row_end, int lane, int L) {
        const int r32 = lane & 31, hi = lane >> 5;
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            const int r = row_begin + t * 32 + r32;
            const bool in = r < row_end;
            const char* src;
            const int i = query_of(p, h, min(r, row_end - 1), src);
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) {
                const int e = kk * 16 + hi * 8;
                q[t][kk] = *(const V8*)(src + min(e, p.d - 8) * 2);
                if (e >= p.d) q[t][kk] = V8{};
            }
            lim[t] = !in ? 0x7fffffff : p.causal ? min(L, max(0, L - p.n + 1 + i)) : L;
            m[t] = kNone;
            l[t] = 0.f;
#pragma unroll
            for (int d = 0; d < D::DVB; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[t][d][e] = 0.f;
        }
    }

    // NS sub-tiles of 32 keys in LDS.  CODES: every key's logits carry its own factor.  masked: some row sees only the keys
    // below its own part's limit (seg), or below P.
    template <int NS, bool CODES>
    __device__ __forceinline__ void tile(const Params& p, const T* kl, const T* vl, const float* scale, int seg, int key0,
                                         bool masked, bool edge, const int* bad, int lane) {
        const int r32 = lane & 31, hi = lane >> 5;
        // Fragments are read one group ahead of the products that take them.  Left alone, the compiler reads each one right
        // before its product and waits out the LDS latency every time (twice the time of a tile); the barriers hold reads and
        // products in this order and let vector instructions pass.
        f32x16 s[QT][NS];
        constexpr int KG = KS == 4 || KS == 8 ? 2 : KS % 4 == 0 ? 4 : KS % 5 == 0 ? 5 : KS, NG = NS * KS / KG;
        V8 kf[2][KG];
        auto read_k = [&](int g) {
#pragma unroll
            for (int i = 0; i < KG; ++i) {
                const int at = g * KG + i, u = at / KS, kk = at - u * KS;
                kf[g & 1][i] = *(const V8*)(kl + (u * 32 + r32) * D::KSTR + kk * 16 + hi * 8);
            }
        };
#pragma unroll
        for (int u = 0; u < NS; ++u)
#pragma unroll
            for (int t = 0; t < QT; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[t][u][e] = 0.f;
        read_k(0);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            if (g + 1 < NG) read_k(g + 1);
            __builtin_amdgcn_sched_barrier(kVector);
#pragma unroll
            for (int i = 0; i < KG; ++i) {
                const int at = g * KG + i, u = at / KS, kk = at - u * KS;
#pragma unroll
                for (int t = 0; t < QT; ++t) s[t][u] = Ops<T>::mfma(kf[g & 1][i], q[t][kk], s[t][u]);
            }
            __builtin_amdgcn_sched_barrier(kVector);
        }
        // Two waves share a SIMD and left alone run in step, both at the products, then both at the softmax.  The one that has its
        // logits goes first until half of its second product is issued; the other one's products then fill the matrix unit
        // beside its exponentials (d = 40, 4 x 4096 queries on 8192 keys: 251 -> 231 us; with 32 rows a wave it gains nothing).
        if (QT == 2) __builtin_amdgcn_s_setprio(1);
        // V^T fragments: lane 16 a + x of a half reads row x / 4, columns 4 (x % 4) .. of a block of 4 keys and 16 columns
        const int x = lane & 15;
        const T* vb = vl + (4 * hi + (x >> 2)) * D::VSTR + ((lane >> 4) & 1) * 16 + (x & 3) * 4;
        V8 vf[2][D::DVB];
        auto read_v = [&](int w) {
#pragma unroll
            for (int d = 0; d < D::DVB; ++d) {
                typedef __attribute__((address_space(3))) s16x4* lds_ptr;
                const T* at = vb + w * 16 * D::VSTR + d * 32;
                const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)at);
                const s16x4 up = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(at + 8 * D::VSTR));
                vf[w & 1][d] = __builtin_bit_cast(V8, __builtin_shufflevector(lo, up, 0, 1, 2, 3, 4, 5, 6, 7));
            }
        };
        const float c = CODES ? 1.f : p.c;
        if (CODES) {
#pragma unroll
            for (int u = 0; u < NS; ++u)
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const float4 f = *(const float4*)(scale + u * 32 + 2 * e + 4 * hi);
#pragma unroll
                    for (int t = 0; t < QT; ++t) { s[t][u][e] *= f.x; s[t][u][e + 1] *= f.y; s[t][u][e + 2] *= f.z; s[t][u][e + 3] *= f.w; }
                }
        }
        if (masked) {
#pragma unroll
            for (int u = 0; u < NS; ++u)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int key = u * 32 + 8 * (e >> 2) + 4 * hi + (e & 3);
                    const bool poison = edge && bad[key];
#pragma unroll
                    for (int t = 0; t < QT; ++t) {
                        if (poison) s[t][u][e] = __builtin_nanf("");
                        if (key0 + key >= (seg ? lim[t] : p.P)) s[t][u][e] = kNegInf;
                    }
                }
        }
        read_v(0);
        V8 pr[QT][NS][2];
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            float mt = s[t][0][0];
#pragma unroll
            for (int u = 0; u < NS; ++u)
#pragma unroll
                for (int e = 0; e < 16; ++e) mt = fmaxf(mt, s[t][u][e]);
            const float2 halves = both_halves(mt);
            mt = fmaxf(halves.x, halves.y) * c;
            // the reference moves only when a logit exceeds it by 2^8: probabilities stay below that, nothing overflows
            const bool up = mt - m[t] > 8.f;
            if (__any(up)) {
                const float mn = up ? mt : m[t];
                const float alpha = __builtin_amdgcn_exp2f(m[t] - mn);
                m[t] = mn;
                l[t] *= alpha;
#pragma unroll
                for (int d = 0; d < D::DVB; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[t][d][e] *= alpha;
            }
            const float off = Ops<T>::kBias - m[t];
#pragma unroll
            for (int u = 0; u < NS; ++u) {
#pragma unroll
                for (int e = 0; e < 16; ++e) s[t][u][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][u][e], c, off));
                if (!ONES)
#pragma unroll
                    for (int e = 0; e < 16; ++e) l[t] += s[t][u][e];
#pragma unroll
                for (int e = 0; e < 16; ++e) pr[t][u][e >> 3][e & 7] = (T)s[t][u][e];
            }
        }
#pragma unroll
        for (int w = 0; w < 2 * NS; ++w) {
            if (QT == 2 && w == NS) __builtin_amdgcn_s_setprio(0);
            if (w + 1 < 2 * NS) read_v(w + 1);
            __builtin_amdgcn_sched_barrier(kVector);
#pragma unroll
            for (int d = 0; d < D::DVB; ++d)
#pragma unroll
                for (int t = 0; t < QT; ++t) o[t][d] = Ops<T>::mfma(vf[w & 1][d], pr[t][w >> 1][w & 1], o[t][d]);
            __builtin_amdgcn_sched_barrier(kVector);
        }
    }

    __device__ __forceinline__ float row_sum(const Params& p, int t) const {
        float sum = l[t];
        if (ONES) {
            // column d of V: block d / 32, register 4 ((d % 32) / 8), lower half (d is a multiple of 8)
#pragma unroll
            for (int d = 0; d < D::DVB; ++d)
#pragma unroll
                for (int e = 0; e < 16; e += 4) sum = d * 32 + 2 * e == p.d ? o[t][d][e] : sum;
            return both_halves(sum).x;
        }
        const float2 halves = both_halves(sum);
        return halves.x + halves.y;
    }
    __device__ __forceinline__ float reference(const Params& p, int t) const { return m[t] == kNone ? kNegInf : m[t] - Ops<T>::kBias; }
    // f(column, four values from there on) for this lane's share of row t
    template <typename F>
    __device__ __forceinline__ void each4(const Params& p, int t, int lane, F f) const {
#pragma unroll
        for (int d = 0; d < D::DVB; ++d)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int c = d * 32 + 2 * e + 4 * (lane >> 5);
                if (c < p.d) f(c, o[t][d][e], o[t][d][e + 1], o[t][d][e + 2], o[t][d][e + 3]);
            }
    }
};

// The same for one tile of 16 queries with heads wider than 128.  Lane 16 g + x holds query x; of the 32 keys of a tile it
// has the logits of keys 4 g .. 4 g + 3 and 16 + 4 g .. 16 + 4 g + 3.
template <typename T, int KS, int QT, bool ONES>
struct Rows16 {
    using D = Dims<KS>;
    using V8 = typename Ops<T>::V8;
    static constexpr int KB = KS / 2, DB = KS;
    V8 q[KB];
    f32x4 o[DB];
    float m[1], l;
    int lim[1];

    __device__ __forceinline__ void init(const Params& p, int h, int row_begin, int row_end, int lane, int L) {
        const int g = lane >> 4, r = row_begin + (lane & 15);
        const char* src;
        const int i = query_of(p, h, min(r, row_end - 1), src);
#pragma unroll
        for (int kk = 0; kk < KB; ++kk) {
            const int e = kk * 32 + g * 8;
            q[kk] = *(const V8*)(src + min(e, p.d - 8) * 2);
            if (e >= p.d) q[kk] = V8{};
        }
        lim[0] = r >= row_end ? 0x7fffffff : p.causal ? min(L, max(0, L - p.n + 1 + i)) : L;
        m[0] = kNone;
        l = 0.f;
#pragma unroll
        for (int d = 0; d < DB; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    template <int NS, bool CODES>
    __device__ __forceinline__ void tile(const Params& p, const T* kl, const T* vl, const float* scale, int seg, int key0,
                                         bool masked, bool edge, const int* bad, int lane) {
        const int x = lane & 15, g = lane >> 4;
        f32x4 s[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < KB; ++kk)
#pragma unroll
            for (int u = 0; u < 2; ++u)
                s[u] = Ops<T>::mfma(*(const V8*)(kl + (u * 16 + x) * D::KSTR + kk * 32 + g * 8), q[kk], s[u]);
        const float c = CODES ? 1.f : p.c;
        if (CODES)
#pragma unroll
            for (int u = 0; u < 2; ++u) s[u] *= *(const f32x4*)(scale + u * 16 + 4 * g);
        if (masked) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int key = u * 16 + 4 * g + e;
                    if (edge && bad[key]) s[u][e] = __builtin_nanf("");
                    if (key0 + key >= (seg ? lim[0] : p.P)) s[u][e] = kNegInf;
                }
        }
        float mt = s[0][0];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) mt = fmaxf(mt, s[u][e]);
        float2 two = both_rows(mt);
        two = both_halves(fmaxf(two.x, two.y));
        mt = fmaxf(two.x, two.y) * c;
        const bool up = mt - m[0] > 8.f;
        if (__any(up)) {
            const float mn = up ? mt : m[0], alpha = __builtin_amdgcn_exp2f(m[0] - mn);
            m[0] = mn;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] *= alpha;
        }
        const float off = Ops<T>::kBias - m[0];
        V8 pr;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][e], c, off));
                l += w;
                pr[4 * u + e] = (T)w;
            }
        typedef __attribute__((address_space(3))) s16x4* lds_ptr;
        const T* vb = vl + (4 * g + (x >> 2)) * D::VSTR + (x & 3) * 4;
#pragma unroll
        for (int d = 0; d < DB; ++d) {
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(vb + d * 16));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(vb + d * 16 + 16 * D::VSTR));
            o[d] = Ops<T>::mfma(__builtin_bit_cast(V8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7)), pr, o[d]);
        }
    }

    __device__ __forceinline__ float row_sum(const Params&, int) const {
        float2 two = both_rows(l);
        two = both_halves(two.x + two.y);
        return two.x + two.y;
    }
    __device__ __forceinline__ float reference(const Params& p, int) const { return m[0] == kNone ? kNegInf : m[0] - Ops<T>::kBias; }
    template <typename F>
    __device__ __forceinline__ void each4(const Params& p, int, int lane, F f) const {
#pragma unroll
        for (int d = 0; d < DB; ++d) {
            const int c = d * 16 + 4 * (lane >> 4);
            if (c < p.d) f(c, o[d][0], o[d][1], o[d][2], o[d][3]);
        }
    }
};

template <typename T, int KS, int QT, bool ONES>
using Rows = typename std::conditional<Dims<KS>::kWide, Rows16<T, KS, QT, ONES>, Rows32<T, KS, QT, ONES>>::type;

template <typename T>
__device__ __forceinline__ void store4(char* p, float a, float b, float c, float d) {
    typedef __attribute__((ext_vector_type(4))) T T4;
    T4 v;
    v[0] = (T)a; v[1] = (T)b; v[2] = (T)c; v[3] = (T)d;
    *(T4*)p = v;
}

struct Item { int h, b, row_begin, row_end, L, TP, v0, v1, slot, per_image; };

// Key range of the item in tiles of KT keys: first the prefix's, then the own ones.
__device__ __forceinline__ bool find_item(const Params& p, Item& it, bool& keys_way) {
    const bool second = (int)blockIdx.x >= p.blocks0;
    const Group& g = p.g[second];
    const int i = (int)blockIdx.x - (second ? p.blocks0 : 0), share = (g.items + kXcd - 1) / kXcd;
    // workgroup i runs on XCD i mod 8: every XCD takes a contiguous share of the items, which share keys through its L2
    int w = (i % kXcd) * share + i / kXcd;
    if (w >= g.items || i / kXcd >= share) return false;
    keys_way = g.keys_way;
    it.per_image = g.per_image;
    int q = g.by_tiles(w);
    const int tile = w - q * g.tiles;
    w = q;
    q = g.by_splits(w);
    const int split = w - q * g.splits;
    it.h = g.per_image ? p.by_B(q) : q;
    it.b = g.per_image ? q - it.h * p.B : 0;
    const int rows = p.n * p.G, first = g.per_image ? it.b * rows : 0, last = g.per_image ? first + rows : p.B * rows;
    it.row_begin = first + tile * g.tile_rows;
    it.row_end = min(last, it.row_begin + g.tile_rows);
    const int KT = g.keys_way ? 32 : 64;
    it.TP = (g.segs & 1) ? (p.P + KT - 1) / KT : 0;
    it.L = 0;
    int TO = 0;
    if (g.segs & 2) {
        it.L = p.own_len ? min(max(p.own_len[it.b], 0), p.S) : p.S;
        int most = it.L;
        if (p.causal) most = min(most, max(0, it.L - p.n + 1 + p.by_G(it.row_end - 1 - first)));
        TO = (most + KT - 1) / KT;
    }
    const long long TT = it.TP + TO;
    it.v0 = (int)(TT * split / g.splits);
    it.v1 = (int)(TT * (split + 1) / g.splits);
    it.slot = g.slot0 + split;
    return true;
}

// What staging never writes: zeros behind head_dim in the rows of K and V, a one in V's spare column.  Two threads a row.
template <typename T, int KS, bool ONES>
__device__ __forceinline__ void clear_pads(const Params& p, T* kl, T* vl, int row, int half) {
    using D = Dims<KS>;
    for (int c = p.d + 8 * half; c < KS * 16; c += 16) *(u32x4*)(kl + row * D::KSTR + c) = u32x4{0u, 0u, 0u, 0u};
    for (int c = p.d + 8 * half; c < D::DVB * 32; c += 16)
        *(u32x4*)(vl + row * D::VSTR + c) = u32x4{ONES && c == p.d ? Ops<T>::kOne : 0u, 0u, 0u, 0u};
}

__device__ __forceinline__ long long out_row(const Params& p, int h, int r) {
    const int tok = p.by_G(r), g = r - tok * p.G;
    return (long long)tok * p.Hq + h * p.G + g;
}

// The query that the item's first row belongs to
__device__ __forceinline__ int item_query(const Params& p, const Item& it) {
    const int tok = p.by_G(it.row_begin);
    return tok - p.by_n(tok) * p.n;
}

template <typename T, int KS, int QT, bool ONES, int FMT>
__device__ __forceinline__ void rows_way(const Params& p, const Item& it, char* lds) {
    constexpr bool CODES = FMT != SID_KV_NONE;
    using D = Dims<KS>;
    using S = Stager<T, KS, 256, 64, FMT>;
    T* kl = (T*)lds;
    T* vl = kl + D::KELEMS;
    float* scales = (float*)(lds + D::kRowData);
    int* flags = (int*)(scales + 128);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wave_row = it.row_begin + wave * D::ROWS * QT;
    // own keys that every row of the item sees: the first row's (in causal order rows see ever more)
    const int least = p.causal ? min(it.L, max(0, it.L - p.n + 1 + item_query(p, it))) : it.L;
    S st;
    Rows<T, KS, QT, ONES> R;
    int seg = it.v0 >= it.TP, t = seg ? it.v0 - it.TP : it.v0, t1 = seg ? it.v1 - it.TP : min(it.v1, it.TP);
    Stream s(p, seg, it.b, it.h, seg ? it.L : p.P);
    if (S::kAhead && t < t1) st.load(p, s, t * 64, tid);
    R.init(p, it.h, wave_row, it.row_end, lane, it.L);                            // while the first tile is on its way
    clear_pads<T, KS, ONES>(p, kl, vl, tid & 127, tid >> 7);
    // With 32 rows a wave the same by workgroup: of the two on a CU (i and i + 256) the later goes first (d = 128: 586 -> 574 us;
    // five tokens of 16 sequences on codes 33.0 -> 32.1).  Not where 16-bit keys stream past the rows of all images (one token
    // of 32 sequences 44.3 -> 45.5), nor above d = 128, where it changes nothing.
    if (QT == 1 && !D::kWide && (CODES || it.per_image) && (blockIdx.x >> 8 & 1)) __builtin_amdgcn_s_setprio(1);
    int buf = 0;
    for (;;) {
        const int seen = seg ? least : p.P;              // tiles that end before it need no mask
        for (; t < t1; ++t) {
            const int key0 = t * 64;
            const bool masked = key0 + 64 > seen, edge = masked && p.causal && seg;
            if (edge) {
                if (tid < 64) flags[buf + tid] = 0;
                __syncthreads();
            }
            if (!S::kAhead) st.load_k(p, s, key0, tid);
            st.store_k(p, kl + buf * D::KSTR, scales + buf, tid);
            if (!S::kAhead) st.load_v(p, s, key0, tid);
            st.store_v(p, vl + buf * D::VSTR, edge, flags + buf, tid);
            __syncthreads();                             // also: every wave is done with the other buffer
            if (S::kAhead && t + 1 < t1) st.load(p, s, key0 + 64, tid);
#pragma unroll
            for (int u = 0; u < 64; u += 32 * D::NS)
                R.template tile<D::NS, CODES>(p, kl + (buf + u) * D::KSTR, vl + (buf + u) * D::VSTR, scales + buf + u, seg, key0 + u,
                                              masked, edge, flags + buf + u, lane);
            buf ^= 64;
        }
        if (seg || it.v1 <= it.TP) break;
        seg = 1;                                         // on to the own keys
        t = 0;
        t1 = it.v1 - it.TP;
        s = Stream(p, 1, it.b, it.h, it.L);
        if (S::kAhead) st.load(p, s, 0, tid);
    }

#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const int r = wave_row + t * D::ROWS + lane % D::ROWS;
        const float sum = R.row_sum(p, t);
        if (r >= it.row_end) continue;
        const long long row = out_row(p, it.h, r);
        if (p.part) {
            const long long at = (long long)it.slot * p.B * p.n * p.Hq + row;
            if (lane < D::ROWS) p.stats[at] = make_float2(R.reference(p, t), sum);
            float* dst = p.part + at * p.d;
            R.each4(p, t, lane, [&](int c, float w, float x, float y, float z) { *(float4*)(dst + c) = make_float4(w, x, y, z); });
        } else {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            char* dst = p.out + row * p.d * 2;
            R.each4(p, t, lane, [&](int c, float w, float x, float y, float z) { store4<T>(dst + c * 2, w * inv, x * inv, y * inv, z * inv); });
        }
    }
}

// Orders one wave's LDS writes before its lanes' reads of one another's (the hardware keeps a wave's LDS operations in
// order; this keeps the compiler from moving them).
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

template <typename T, int KS, bool ONES, int FMT>
__device__ __forceinline__ void keys_way(const Params& p, const Item& it, char* lds) {
    constexpr bool CODES = FMT != SID_KV_NONE;
    using D = Dims<KS>;
    using S = Stager<T, KS, 64, 32, FMT>;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), buf = wave * 32;
    T *k = (T*)lds + buf * D::KSTR, *v = (T*)lds + D::KELEMS + buf * D::VSTR;             // this wave's own rows
    float* scales = (float*)(lds + D::kRowData) + buf;
    int* flags = (int*)(lds + D::kRowData) + 128 + buf;
    const int least = p.causal ? min(it.L, max(0, it.L - p.n + 1 + item_query(p, it))) : it.L;
    S st;
    Rows<T, KS, 1, ONES> R;
    // the groups of few-row items have one part each (make_plan)
    const int seg = it.TP == 0, t1 = it.v1, seen = seg ? least : p.P;
    int t = it.v0 + wave;
    const Stream s(p, seg, it.b, it.h, seg ? it.L : p.P);
    if (S::kAhead && t < t1) st.load(p, s, t * 32, lane);
    R.init(p, it.h, it.row_begin, it.row_end, lane, it.L);
    clear_pads<T, KS, ONES>(p, k, v, lane & 31, lane >> 5);
    for (; t < t1; t += 4) {
        const int key0 = t * 32;
        const bool masked = key0 + 32 > seen, edge = masked && p.causal && seg;
        wave_sync();                                     // the last tile's reads come before this one's writes
        if (edge) {
            if (lane < 32) flags[lane] = 0;
            wave_sync();
        }
        if (!S::kAhead) st.load_k(p, s, key0, lane);
        st.store_k(p, k, scales, lane);
        if (!S::kAhead) st.load_v(p, s, key0, lane);
        st.store_v(p, v, edge, flags, lane);
        wave_sync();
        if (S::kAhead && t + 4 < t1) st.load(p, s, key0 + 128, lane);
        R.template tile<1, CODES>(p, k, v, scales, seg, key0, masked, edge, flags, lane);
    }

    const float sum = R.row_sum(p, 0);
    __syncthreads();
    float* jo = (float*)lds;                             // [4][32][MSTR], then references and sums [4][32]
    float* jm = jo + 4 * 32 * D::MSTR;
    float* jl = jm + 128;
    if (lane < D::ROWS) { jm[buf + lane] = R.reference(p, 0); jl[buf + lane] = sum; }
    float* mine = jo + (buf + lane % D::ROWS) * D::MSTR;
    R.each4(p, 0, lane, [&](int c, float a, float x, float y, float z) { *(float4*)(mine + c) = make_float4(a, x, y, z); });
    __syncthreads();
    const int rr = tid >> 3, r = it.row_begin + rr;      // 8 threads per row
    if (rr >= D::ROWS || r >= it.row_end) return;
    float top = kNegInf, w[4], total = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) top = fmaxf(top, jm[k * 32 + rr]);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        w[k] = jm[k * 32 + rr] == kNegInf ? 0.f : __builtin_amdgcn_exp2f(jm[k * 32 + rr] - top);
        total = __builtin_fmaf(w[k], jl[k * 32 + rr], total);
    }
    // a wave whose keys gave NaN has no finite reference but a NaN sum
#pragma unroll
    for (int k = 0; k < 4; ++k) if (!(jl[k * 32 + rr] == jl[k * 32 + rr])) total = __builtin_nanf("");
    const long long row = out_row(p, it.h, r);
    const long long at = (long long)it.slot * p.B * p.n * p.Hq + row;
    const float inv = total == 0.f ? 0.f : 1.f / total;
    if (p.part && (tid & 7) == 0) p.stats[at] = make_float2(top, total);
    for (int c = (tid & 7) * 4; c < p.d; c += 32) {
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float4 o = *(const float4*)(jo + (k * 32 + rr) * D::MSTR + c);
            a.x = __builtin_fmaf(w[k], o.x, a.x); a.y = __builtin_fmaf(w[k], o.y, a.y);
            a.z = __builtin_fmaf(w[k], o.z, a.z); a.w = __builtin_fmaf(w[k], o.w, a.w);
        }
        if (p.part) *(float4*)(p.part + at * p.d + c) = a;
        else store4<T>(p.out + (row * p.d + c) * 2, a.x * inv, a.y * inv, a.z * inv, a.w * inv);
    }
}

// QT > 1: items share rows only (many rows per image); QT == 1: either way, by the item's group.
template <typename T, int KS, int QT, bool ONES, int FMT>
__global__ void __launch_bounds__(256, KS <= 8 ? 2 : 1) shared_kernel(Params p) {
    extern __shared__ __align__(16) char lds[];
    Item it;
    bool by_keys;
    if (!find_item(p, it, by_keys)) return;
    if (QT == 1 && by_keys) keys_way<T, KS, ONES, FMT>(p, it, lds);
    else rows_way<T, KS, QT, ONES, FMT>(p, it, lds);
}

template <typename T, int KS, int QT, bool ONES, int FMT>
int launch(const Params& p, unsigned grid, hipStream_t st) {
    using D = Dims<KS>;
    if (int rc = sid::allow_dynamic_lds<shared_kernel<T, KS, QT, ONES, FMT>>(D::kLds)) return rc;
    hipLaunchKernelGGL((shared_kernel<T, KS, QT, ONES, FMT>), dim3(grid), dim3(256), D::kLds, st, p);
    SID_CHECK_HIP(hipGetLastError());
    return SID_OK;
}

// Classes of head_dim by KS; a head_dim that fills V's last block of 32 leaves no spare column for the row sum.
constexpr int kClasses[6] = {3, 4, 5, 8, 10, 16};
inline int class_of(int d) {
    for (int ks : kClasses) if (d <= ks * 16) return ks;
    return 0;
}
constexpr bool two_tiles(int ks) { return ks <= 4; }      // 64 rows per wave fit in the registers
constexpr int tile_rows(int ks) { return ks <= 8 ? 32 : 16; }

template <typename T, int FMT>
int launch_type(const Params& p, int qt, unsigned grid, hipStream_t st) {
    const bool ones = p.d < 32 * ((class_of(p.d) + 1) / 2);
    switch (class_of(p.d)) {
        case 3: return qt == 2 ? launch<T, 3, 2, true, FMT>(p, grid, st) : launch<T, 3, 1, true, FMT>(p, grid, st);
        case 4:
            if (ones) return qt == 2 ? launch<T, 4, 2, true, FMT>(p, grid, st) : launch<T, 4, 1, true, FMT>(p, grid, st);
            return qt == 2 ? launch<T, 4, 2, false, FMT>(p, grid, st) : launch<T, 4, 1, false, FMT>(p, grid, st);
        case 5: return launch<T, 5, 1, true, FMT>(p, grid, st);
        case 8: return ones ? launch<T, 8, 1, true, FMT>(p, grid, st) : launch<T, 8, 1, false, FMT>(p, grid, st);
        case 10: return launch<T, 10, 1, false, FMT>(p, grid, st);
        default: return launch<T, 16, 1, false, FMT>(p, grid, st);
    }
}

// One unit each: bf16 and f16, parts of 16-bit numbers and parts of codes.
int launch_bf16(const Params& p, int qt, unsigned grid, hipStream_t st);
int launch_f16(const Params& p, int qt, unsigned grid, hipStream_t st);
int launch_bf16_codes(const Params& p, int fmt, int qt, unsigned grid, hipStream_t st);
int launch_f16_codes(const Params& p, int fmt, int qt, unsigned grid, hipStream_t st);

}  // namespace sid_shared
