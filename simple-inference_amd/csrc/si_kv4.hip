// si_kv4.hip -- the K/V cache held in 4 bits: RoPE + quantize + append, fp16
// rows in and out, and GQA attention over its pages; and page copies.  The
// reference keeps one fp16 cache per layer (qwen_one_layer.c:262-266); none of
// this has a counterpart there.
//
// The block: 32 values x of a K or V row share a scale,
//   m = the value of largest magnitude (the negative one of a pair; NaN as 0)
//   h = fp16(r7(min(max(-m / 128, -508), 508)))   r7: 7 significant bits, to even
//   n = min(max(floor(x / (16 h) + 8.5), 0), 15)  in exact arithmetic; 8 if h = 0
// and x is held as 16 h (n - 8): Q4_0's rule (ggml), whose extreme value takes the
// 16th level, with a scale of 7 bits.  7 bits cost nothing next to 4 (the nibbles
// are rounded with the scale as stored), and buy two exact fp16 values: 72 h' for
// the fused unpacking (64 + n) h' - 72 h' of the V operand (4 + 7 bits), and the
// held value itself (4 + 7 bits, at most 8 * 16 * 508 = 65024): a row read back
// into an fp16 cache is what the 4-bit cache attends to, bit for bit.
//
// A page (page_size positions, a power of two >= 16) holds for each KV head its
// nibbles and then its scales (9/16 byte a value):
//   K nibbles [pos/8][pos/4 % 2][dim/8 % 4][pos % 4][dim/32][dim % 8]
//   V nibbles [pos/8][dim/16 in fours, then the rest][dim % 16][dim/16 % 4][pos % 8]
//   scales    [pos/8][dim/32][pos % 4][pos/4 % 2] fp16
// so that the operand lane (l % 16, l / 16) of a 16x16x32 MFMA finds its K row's
// dims 8 (l / 16) .. + 7 of every block, its V dim's 8 positions, and the scales
// of its 8 positions each as one run of up to 16 bytes.
#include "si_device.hpp"
#include "si_kernels.hpp"

namespace si {

// ---------------------------------------------------------------------------
// layout
// ---------------------------------------------------------------------------
__host__ __device__ constexpr int kv4_head_bytes(int hdim, int page_size) {
    return page_size * hdim / 16 * 9;
}
// byte of the dword with K's dims 8 o .. 8 o + 7 of page position i
__device__ __forceinline__ int kv4_k_dword(int D, int i, int o) {
    return (i >> 3) * 4 * D + ((i >> 2) & 1) * 2 * D + (o & 3) * (D / 2) + (i & 3) * (D / 8) +
           (o >> 2) * 4;
}
// byte of the dword with V's dim e of page positions 8 u .. 8 u + 7
__device__ __forceinline__ int kv4_v_dword(int D, int u, int e) {
    const int dt = e >> 4, n = e & 15, full = D / 64 * 4;
    return u * 4 * D + (dt < full ? (dt >> 2) * 256 + n * 16 + (dt & 3) * 4
                                  : full * 64 + n * 8 + (dt - full) * 4);
}
// byte of the scale of block b of page position i
__device__ __forceinline__ int kv4_scale(int D, int page_size, int i, int b) {
    return page_size * (D / 2) + ((i >> 3) * (D / 32) + b) * 16 + (i & 3) * 4 + ((i >> 2) & 1) * 2;
}

__device__ __forceinline__ int Kv4Cache::page_of(int seq, int pos) const {
    const int pg = pages[(size_t)seq * max_pages + min(pos >> shift, max_pages - 1)];
    return min(max(pg, 0), npages - 1);
}

// ---------------------------------------------------------------------------
// the block's quantization
// ---------------------------------------------------------------------------
// Orders values by magnitude, the negative one of a pair above (unsigned); NaN
// must be gone.
__device__ __forceinline__ uint32_t kv4_key(float x) {
    const uint32_t u = f2u(x);
    return u << 1 | u >> 31;
}

// h (as fp16 bits) of the block whose largest key is `key`
__device__ __forceinline__ uint16_t kv4_scale_of(uint32_t key) {
    const float m = u2f(key >> 1 | key << 31);
    const float t = __builtin_amdgcn_fmed3f(__fmul_rn(m, -0.0078125f), -508.0f, 508.0f);
    uint32_t u = f2u(t);
    u = (u + 0xffffu + ((u >> 17) & 1u)) & ~0x1ffffu;
    return __builtin_bit_cast(uint16_t, (_Float16)u2f(u));
}

struct Kv4Scale {
    float a, inv;   // |16 h|, about 1 / a
    uint32_t sign;  // of h
    bool zero;
    __device__ __forceinline__ explicit Kv4Scale(uint16_t h) {
        const float d = h2f_fast(h) * 16.0f;
        a = fabsf(d);
        sign = f2u(d) & 0x80000000u;
        zero = d == 0.0f;
        inv = __builtin_amdgcn_rcpf(a);
    }
    // n of x: the largest n with (n - 8.5) a <= x's side of h, in 0..15.  The
    // estimate is at most one step off; the border products (5 + 7 bits) are
    // exact, so the comparisons decide as exact arithmetic would.
    __device__ __forceinline__ uint32_t nibble(float x) const {
        const float y = u2f(f2u(x) ^ sign);
        float n = __builtin_amdgcn_fmed3f(floorf(fmaf(y, inv, 8.5f)), 0.0f, 15.0f);
        if (y < (n - 8.5f) * a) n -= 1.0f;
        if (y >= (n - 7.5f) * a) n += 1.0f;
        return zero ? 8u : (uint32_t)(int)__builtin_amdgcn_fmed3f(n, 0.0f, 15.0f);
    }
};

// Which tokens of a call fall into a workgroup's unit, 8 positions aligned at 8
// of one sequence: with pos_step 1 the call's tokens are positions pos0 + t of
// sequence 0, else token t is one position of sequence t (ctx_dev[t] - 1, or
// pos0).  Tokens t0 + j sit at base + j for j in [lo, hi).
struct Kv4Unit {
    int seq, base, t0, lo, hi;
    __device__ __forceinline__ Kv4Unit(int x, int ntok, int pos0, int pos_step,
                                       const int *ctx_dev, int limit) {
        if (pos_step) {
            seq = 0;
            base = (pos0 & ~7) + 8 * x;
            t0 = base - pos0;
            lo = max(-t0, 0);
            hi = min(min(ntok - t0, limit - base), 8);
        } else {
            const int ctx = ctx_dev ? ctx_dev[x] : pos0 + 1;
            const bool live = ctx >= 1 && ctx <= limit;  // device contexts: not host-checked
            const int pos = live ? ctx - 1 : 0;
            seq = x;
            base = pos & ~7;
            lo = pos & 7;
            t0 = x - lo;
            hi = live ? lo + 1 : lo;
        }
    }
};

static int kv4_units(int ntok, int pos0, int pos_step) {
    return pos_step ? (int)(((long long)pos0 + ntok + 7) / 8 - pos0 / 8) : ntok;
}

// ---------------------------------------------------------------------------
// append: block of 2 D threads per (unit, KV head), then blocks that rotate q.
// K: thread (position, octet of dims), a block's four octets in a quad of lanes.
// V: thread per dim with the unit's 8 positions, a block in 32 lanes; a dword
// whose 8 positions are not all written keeps its other nibbles.
// HALF_IN: the rows are fp16 cache rows (kin, vin), copied in without RoPE.
// ---------------------------------------------------------------------------
template <int D, bool HALF_IN>
__global__ void __launch_bounds__(2 * D) k_kv4_append(
    const float *__restrict__ qkv, int ldqkv, const uint16_t *__restrict__ kin,
    const uint16_t *__restrict__ vin, int qheads, int ntok, int pos0, int pos_step, int limit,
    const int *__restrict__ ctx_dev, const float *__restrict__ rc, const float *__restrict__ rs,
    float *__restrict__ q_out, Kv4Cache c) {
    constexpr int HALF = D / 2;
    const Kv4Unit un((int)blockIdx.x, ntok, pos0, pos_step, ctx_dev, limit);
    if (un.lo >= un.hi) return;
    const int tid = threadIdx.x, kvh = c.kvheads, qd = qheads * D, kvd = kvh * D;
    const int g = blockIdx.y;
    if (!HALF_IN && g >= kvh) {
        const int i0 = ((g - kvh) * 2 * D + tid);  // pair index over the q heads
        if (i0 >= qd / 2) return;
        const int h = i0 / HALF, i = i0 % HALF;
        for (int j = un.lo; j < un.hi; ++j) {
            const int t = un.t0 + j;
            const float cs = rc[(size_t)(un.base + j) * HALF + i];
            const float sn = rs[(size_t)(un.base + j) * HALF + i];
            const float *row = qkv + (size_t)t * ldqkv + h * D;
            const float a = row[i], b = row[i + HALF];
            float *qo = q_out + (size_t)t * qd + h * D;
            qo[i] = __fsub_rn(__fmul_rn(a, cs), __fmul_rn(b, sn));
            qo[i + HALF] = __fadd_rn(__fmul_rn(b, cs), __fmul_rn(a, sn));
        }
        return;
    }
    const int page_size = 1 << c.shift;
    const size_t at = ((size_t)c.page_of(un.seq, un.base) * kvh + g) *
                      (size_t)kv4_head_bytes(D, page_size);
    const int in_page = un.base & (page_size - 1);
    if (tid < D) {
        uint8_t *kp = c.k + at;
        const int j = tid / (D / 8), o = tid % (D / 8), pos = un.base + j, i = in_page + j;
        const bool live = j >= un.lo && j < un.hi;
        float x[8];
        uint32_t key = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float v = 0.0f;
            if (live) {
                const int dim = 8 * o + e;
                if constexpr (HALF_IN) {
                    v = h2f_fast(kin[(size_t)(un.t0 + j) * kvd + g * D + dim]);
                } else {
                    const float *row = qkv + (size_t)(un.t0 + j) * ldqkv + qd + g * D;
                    const int ii = dim < HALF ? dim : dim - HALF;
                    const float cs = rc[(size_t)pos * HALF + ii], sn = rs[(size_t)pos * HALF + ii];
                    const float a = row[ii], b = row[ii + HALF];
                    v = dim < HALF ? __fsub_rn(__fmul_rn(a, cs), __fmul_rn(b, sn))
                                   : __fadd_rn(__fmul_rn(b, cs), __fmul_rn(a, sn));
                }
            }
            x[e] = v == v ? v : 0.0f;
            key = max(key, kv4_key(x[e]));
        }
        key = max(key, (uint32_t)dpp_i<DPP_XOR1>((int)key));
        key = max(key, (uint32_t)dpp_i<DPP_XOR2>((int)key));
        const uint16_t h = kv4_scale_of(key);
        const Kv4Scale sc(h);
        uint32_t w = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) w |= sc.nibble(x[e]) << (4 * e);
        if (live) {
            *(uint32_t *)(kp + kv4_k_dword(D, i, o)) = w;
            if ((o & 3) == 0) *(uint16_t *)(kp + kv4_scale(D, page_size, i, o >> 2)) = h;
        }
    } else {
        uint8_t *vp = c.v + at;
        const int e = tid - D;
        uint32_t w = 0, mask = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const bool live = j >= un.lo && j < un.hi;
            float v = 0.0f;
            if (live) {
                if constexpr (HALF_IN) v = h2f_fast(vin[(size_t)(un.t0 + j) * kvd + g * D + e]);
                else v = qkv[(size_t)(un.t0 + j) * ldqkv + qd + kvd + g * D + e];
            }
            v = v == v ? v : 0.0f;
            uint32_t key = kv4_key(v);
            key = max(key, (uint32_t)dpp_i<DPP_XOR1>((int)key));
            key = max(key, (uint32_t)dpp_i<DPP_XOR2>((int)key));
            key = max(key, (uint32_t)dpp_i<DPP_ROR4>((int)key));
            key = max(key, (uint32_t)dpp_i<DPP_ROR8>((int)key));
            key = max(key, (uint32_t)swap16_i((int)key));
            const uint16_t h = kv4_scale_of(key);
            w |= Kv4Scale(h).nibble(v) << (4 * j);
            mask |= live ? 15u << (4 * j) : 0u;
            if (live && (e & 31) == 0)
                *(uint16_t *)(vp + kv4_scale(D, page_size, in_page + j, e >> 5)) = h;
        }
        uint32_t *dst = (uint32_t *)(vp + kv4_v_dword(D, in_page >> 3, e));
        *dst = mask == 0xffffffffu ? w : (*dst & ~mask) | (w & mask);
    }
}

// ---------------------------------------------------------------------------
// rows back as fp16, exactly: the same units, a thread per (position, octet) of
// K and per dim of V
// ---------------------------------------------------------------------------
template <int D>
__global__ void __launch_bounds__(2 * D) k_kv4_read(Kv4Cache c, int ntok, int pos0, int pos_step,
                                                    int limit, const int *__restrict__ ctx_dev,
                                                    uint16_t *__restrict__ kout,
                                                    uint16_t *__restrict__ vout) {
    const Kv4Unit un((int)blockIdx.x, ntok, pos0, pos_step, ctx_dev, limit);
    if (un.lo >= un.hi) return;
    const int tid = threadIdx.x, kvh = c.kvheads, kvd = kvh * D, g = blockIdx.y;
    const int page_size = 1 << c.shift;
    const size_t at = ((size_t)c.page_of(un.seq, un.base) * kvh + g) *
                      (size_t)kv4_head_bytes(D, page_size);
    const int in_page = un.base & (page_size - 1);
    if (tid < D) {
        const uint8_t *kp = c.k + at;
        const int j = tid / (D / 8), o = tid % (D / 8), i = in_page + j;
        if (j < un.lo || j >= un.hi) return;
        const uint32_t w = *(const uint32_t *)(kp + kv4_k_dword(D, i, o));
        const float d = h2f_fast(*(const uint16_t *)(kp + kv4_scale(D, page_size, i, o >> 2))) * 16.0f;
        uint16_t y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
            y[e] = __builtin_bit_cast(uint16_t, (_Float16)((float)((int)(w >> (4 * e) & 15) - 8) * d));
        *(uint4 *)(kout + (size_t)(un.t0 + j) * kvd + g * D + 8 * o) = *(const uint4 *)y;
    } else {
        const uint8_t *vp = c.v + at;
        const int e = tid - D;
        const uint32_t w = *(const uint32_t *)(vp + kv4_v_dword(D, in_page >> 3, e));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (j < un.lo || j >= un.hi) continue;
            const float d =
                h2f_fast(*(const uint16_t *)(vp + kv4_scale(D, page_size, in_page + j, e >> 5))) * 16.0f;
            vout[(size_t)(un.t0 + j) * kvd + g * D + e] =
                __builtin_bit_cast(uint16_t, (_Float16)((float)((int)(w >> (4 * j) & 15) - 8) * d));
        }
    }
}

// ---------------------------------------------------------------------------
// attention over the pages: a workgroup per (context chunk, KV head, query), its
// four wavefronts take every fourth group of 32 positions.  Per group
//     S^T[pos][head] = K[pos][:] . q[head][:]        (v_mfma_f32_16x16x32_f16)
//     O^T[dim][head] += V^T[dim][pos] . P[pos][head]
// with the group's two score tiles' rows placed so that lane (col, g) gets the
// scores of positions 8 g .. 8 g + 7 in registers, which is the k-slice its lane
// supplies of P: nothing moves between lanes.
//
// K: a masked nibble is the fp16 subnormal n 2^-24 (or 16 n 2^-24 in the odd
// places, where q carries 1/16), which the matrix cores take exactly: 5 operations
// unpack 8 values.  -8 sum q is the product's C operand, the block's scale
// multiplies the 16x16 result (4 operations a block and lane against 8 values').
// V: (64 + n) h - 72 h in one fused operation a pair, exact in fp16 (above).
//
// q and the weights go in as fp16 hi + lo pairs.  q's are integers of a common
// unit, 12 bits each of the head's largest value: every sum of 32 products (20
// bits) is then exact in the matrix core, whose own rounding of a sum with an
// offset of 8 sum q would show (24 bits of the head's largest q in all; as
// fp16 roundings of q the result was off by up to 2.7e-5).  The weights' pair
// has 22 bits.  With at most 8 heads a KV head both halves share one product:
// columns 0-7 carry hi, 8-15 lo, and their results are added across (WIDE: 9 to
// 16 heads, two products).
//
// The running maximum is moved only when a score passes it by 2^8 (weights up to
// 256 fit the fp16 pair as well as weights up to 1), a wavefront-uniform branch.
// ---------------------------------------------------------------------------
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int A4_GROUP = 32;             // positions of a wavefront's step
constexpr int A4_STEP = 4 * A4_GROUP;    // of a workgroup's

__device__ __forceinline__ float ror8_add(float v) { return v + dpp_f<DPP_ROR8>(v); }

// N dwords at p, aligned to what N allows
template <int N>
__device__ __forceinline__ void load_dwords(const uint8_t *p, uint32_t (&w)[N]) {
    if constexpr (N == 1) {
        w[0] = *(const uint32_t *)p;
    } else if constexpr (N == 2) {
        const uint2 t = *(const uint2 *)p;
        w[0] = t.x, w[1] = t.y;
    } else if constexpr (N == 3) {
        const uint3 t = *(const uint3 *)p;
        w[0] = t.x, w[1] = t.y, w[2] = t.z;
    } else {
        const uint4 t = *(const uint4 *)p;
        w[0] = t.x, w[1] = t.y, w[2] = t.z, w[3] = t.w;
    }
}

// What a wavefront reads of a group: lane (col, g)'s K nibbles of both tiles, V
// nibbles, and dword col of the D / 8 dwords that hold the scales of positions
// 8 g .. 8 g + 7: all 16 lanes of a row need them all, and take them with a DPP
// broadcast in the row where they are used.
template <int D>
struct Kv4Group {
    static constexpr int KS = D / 32, DT = D / 16;
    uint32_t k[2][KS], v[DT], kh, vh;
    // kk, ks, vv: the KV head's part of the page with the K row's, the K scales'
    // and the V positions' unit; ku, vu: the units' places in it
    __device__ __forceinline__ void load(const uint8_t *kk, int ku, const uint8_t *ks,
                                         const uint8_t *vv, int vu, int nib, int lane) {
        const int r = lane & 15, g = lane >> 4;
        const int so = nib + vu * KS * 16 + min(r, 4 * KS - 1) * 4;
        kh = *(const uint32_t *)(ks + so);
        vh = *(const uint32_t *)(vv + so);
#pragma unroll
        for (int t = 0; t < 2; ++t)
            load_dwords<KS>(kk + ku * 4 * D + t * 2 * D + g * (D / 2) + (r & 3) * (D / 8), k[t]);
        constexpr int FULL = D / 64;
#pragma unroll
        for (int f = 0; f < FULL; ++f) {
            uint32_t w[4];
            load_dwords<4>(vv + vu * 4 * D + f * 256 + r * 16, w);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * f + e] = w[e];
        }
        if constexpr (DT % 4) {
            uint32_t w[2];
            load_dwords<2>(vv + vu * 4 * D + FULL * 256 + r * 8, w);
            v[DT - 2] = w[0], v[DT - 1] = w[1];
        }
    }
};

// lane N of each row of 16 lanes (row_newbcast)
template <int N>
__device__ __forceinline__ uint32_t row_bcast(uint32_t v) {
    return (uint32_t)dpp_i<0x150 + N>((int)v);
}

// the row's dwords 4 b + i as h[b][i]
template <int KS>
__device__ __forceinline__ void spread(uint32_t v, u4 (&h)[KS]) {
    h[0] = (u4){row_bcast<0>(v), row_bcast<1>(v), row_bcast<2>(v), row_bcast<3>(v)};
    if constexpr (KS > 1) h[1] = (u4){row_bcast<4>(v), row_bcast<5>(v), row_bcast<6>(v), row_bcast<7>(v)};
    if constexpr (KS > 2) h[2] = (u4){row_bcast<8>(v), row_bcast<9>(v), row_bcast<10>(v), row_bcast<11>(v)};
    if constexpr (KS > 3) h[3] = (u4){row_bcast<12>(v), row_bcast<13>(v), row_bcast<14>(v), row_bcast<15>(v)};
}

__device__ __forceinline__ h2 as_h2(uint32_t u) { return __builtin_bit_cast(h2, u); }
__device__ __forceinline__ uint32_t as_u(h2 h) { return __builtin_bit_cast(uint32_t, h); }

template <int D, bool WIDE, bool PAGE16>
__global__ void __launch_bounds__(256, 2) k_attn_kv4(
    const float *__restrict__ q, int qheads, Kv4Cache c, const int *__restrict__ ctx_dev, int ctx0,
    int ctx_step, int max_ctx, int chunk, float scale2, float *__restrict__ ws_m,
    float *__restrict__ ws_l, float *__restrict__ ws_o, float *__restrict__ attn,
    int8_t *__restrict__ qs, uint16_t *__restrict__ qd8, int16_t *__restrict__ bsum) {
    constexpr int KS = D / 32, DT = D / 16, COLS = WIDE ? 16 : 8;
    __shared__ __attribute__((aligned(16))) float mo[4][COLS][D];
    __shared__ float mm[4][COLS], ml[4][COLS], sc[COLS][4], linv[COLS];
    const int sp = blockIdx.x, g0 = blockIdx.y, qi = blockIdx.z, ns = gridDim.x;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int per = qheads / c.kvheads, seq = ctx_step ? 0 : qi;
    const int ctx = min(ctx_dev ? ctx_dev[qi] : ctx0 + qi * ctx_step, max_ctx);
    if (ns > 1 && ctx_dev) {
        // shares of the longest context there is
        int most = 0;
        for (int i = lane; i < (int)gridDim.z; i += 64) most = max(most, ctx_dev[i]);
        most = min(__builtin_amdgcn_readfirstlane(wave_max_i(most)), max_ctx);
        chunk = max(((most + ns - 1) / ns + A4_STEP - 1) / A4_STEP, 1) * A4_STEP;
    }
    const int p0 = sp * chunk, p1 = min(ctx, p0 + chunk);
    if (ns > 1 && p0 >= p1) {  // an empty state
        for (int h = tid; h < per; h += 256) {
            const size_t pi = ((size_t)qi * qheads + g0 * per + h) * ns + sp;
            ws_m[pi] = -INFINITY;
            ws_l[pi] = 0.0f;
        }
        return;
    }
    // groups of this wavefront: s0 = p0 + 32 wave, + 128, ...
    const int page_size = 1 << c.shift, nib = page_size * (D / 2);
    const size_t hb = (size_t)kv4_head_bytes(D, page_size);
    const int *pages = c.pages + (size_t)seq * c.max_pages;
    // The page ids are read a step before the loads that need them.
    struct Ids { int a, b; };
    auto ids_of = [&](int s0) {  // (uniform)
        Ids i;
        i.a = pages[min(s0 >> c.shift, c.max_pages - 1)];
        i.b = PAGE16 ? pages[min((s0 >> c.shift) + 1, c.max_pages - 1)] : 0;
        return i;
    };
    auto head_at = [&](int pg) {
        return ((size_t)min(max(pg, 0), c.npages - 1) * c.kvheads + g0) * hb;
    };
    auto load = [&](Kv4Group<D> &t, int s0, Ids id) {
        const size_t a = head_at(id.a);
        if constexpr (PAGE16) {
            // two pages a group: units 0, 1 and 2, 3
            const size_t b = head_at(id.b);
            const size_t ka = (lane & 8) ? b : a, va = (lane & 32) ? b : a;
            t.load(c.k + ka, (lane >> 2) & 1, c.k + va, c.v + va, g & 1, nib, lane);
        } else {
            const int u = (s0 & (page_size - 1)) >> 3;
            t.load(c.k + a, u + ((lane >> 2) & 3), c.k + a, c.v + a, u + g, nib, lane);
        }
    };
    int s0 = p0 + A4_GROUP * wave;
    Kv4Group<D> ta, tb;
    Ids id = ids_of(s0);
    if (s0 < p1) load(ta, s0, id);
    id = ids_of(s0 + A4_STEP);

    // q of the lane's column as the B operand, dims 32 b + 8 g + (0, 4, 1, 5, 2, 6,
    // 3, 7), the odd ones over 16: integers hi and lo, q = (hi + lo 2^-12) 2^(ex - 10)
    h8 qa[KS], qb[WIDE ? KS : 1];
    f4 c8[KS], c8l[WIDE ? KS : 1];
    float fac;
    const float lo_col = !WIDE && col >= 8 ? 1.0f : 0.0f;
    {
        const int hc = WIDE ? col : col & 7;
        const bool live = hc < per;
        const float *row = q + ((size_t)qi * qheads + g0 * per + (live ? hc : 0)) * D + 8 * g;
        float x[KS][8], big = 0.0f;
#pragma unroll
        for (int b = 0; b < KS; ++b)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[b][e] = live ? row[32 * b + e] : 0.0f;
                big = fmaxf(big, fabsf(x[b][e]));
            }
        big = fmaxf(big, swap16_f(big));
        big = fmaxf(big, swap32_f(big));
        const int ex = big == 0.0f ? 0 : (int)(f2u(big) >> 23) - 127;
        // the scores' units: 2^24 of the subnormals, 16 of the scale, q's
        fac = __builtin_amdgcn_ldexpf(scale2, 28 + ex - 10 - (!WIDE && col >= 8 ? 12 : 0));
        const u4 eight = {0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u};  // -8 in them
#pragma unroll
        for (int b = 0; b < KS; ++b) {
            h8 hi, lo;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int dim = (e >> 1) + (e & 1) * 4;
                const float y = __builtin_amdgcn_ldexpf(x[b][dim], 10 - ex), yh = rintf(y);
                const float odd = (dim & 1) ? 0.0625f : 1.0f;
                hi[e] = (_Float16)(yh * odd);
                lo[e] = (_Float16)(rintf((y - yh) * 4096.0f) * odd);
            }
            c8[b] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
            if constexpr (WIDE) {
                qa[b] = hi;
                qb[b] = lo;
                c8l[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, eight), lo,
                                                                c8[b], 0, 0, 0);
            } else {
                const u4 uh = __builtin_bit_cast(u4, hi), ul = __builtin_bit_cast(u4, lo);
                u4 us;
#pragma unroll
                for (int e = 0; e < 4; ++e) us[e] = col >= 8 ? ul[e] : uh[e];
                qa[b] = __builtin_bit_cast(h8, us);
            }
            c8[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, eight), qa[b],
                                                           c8[b], 0, 0, 0);
        }
    }

    float m = -INFINITY, lsum = 0.0f;  // of the column; lsum over the lane's positions
    f4 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = (f4){0.0f, 0.0f, 0.0f, 0.0f};

    auto step = [&](Kv4Group<D> &t, int s) {
        float p[2][4];
        u4 hk[KS];
        spread<KS>(t.kh, hk);
#pragma unroll
        for (int tl = 0; tl < 2; ++tl) {
            f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int b = 0; b < KS; ++b) {
                const uint32_t w = t.k[tl][b], w8 = w >> 8;
                const u4 a = {w & 0x000f000fu, w & 0x00f000f0u, w8 & 0x000f000fu, w8 & 0x00f000f0u};
                const h8 ka = __builtin_bit_cast(h8, a);
                f4 d = c8[b];
                d = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qa[b], d, 0, 0, 0);
                if constexpr (WIDE) {
                    const f4 dl = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qb[b], c8l[b], 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; ++i) d[i] = fmaf(dl[i], 0x1p-12f, d[i]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i] = fmaf((float)as_h2(hk[b][i])[tl], d[i], acc[i]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) p[tl][i] = WIDE ? acc[i] * fac : ror8_add(acc[i] * fac);
        }
        if (s + A4_GROUP > p1) {  // wavefront-uniform: positions past the end
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool l0 = s + 8 * g + i < p1, l1 = s + 8 * g + 4 + i < p1;
                p[0][i] = l0 ? p[0][i] : -INFINITY;
                p[1][i] = l1 ? p[1][i] : -INFINITY;
            }
            // their V scales may be anything: 0 (weight 0 * NaN would stay); dword col
            // holds positions 8 g + col % 4 and 4 further
            const int at = s + 8 * g + (col & 3);
            t.vh &= (at < p1 ? 0xffffu : 0u) | (at + 4 < p1 ? 0xffff0000u : 0u);
        }
        float mx = fmaxf(fmaxf(fmaxf(p[0][0], p[0][1]), fmaxf(p[0][2], p[0][3])),
                         fmaxf(fmaxf(p[1][0], p[1][1]), fmaxf(p[1][2], p[1][3])));
        if (__ballot(mx > m + 8.0f)) {
            mx = fmaxf(mx, swap16_f(mx));
            mx = fmaxf(mx, swap32_f(mx));
            const float mn = fmaxf(m, mx);
            const float al = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            lsum *= al;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[dt] *= al;
        }
        u4 pa, pb;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = __builtin_amdgcn_exp2f(p[0][i] - m), y = __builtin_amdgcn_exp2f(p[1][i] - m);
            lsum += x + y;
            const h2 hi = {(_Float16)x, (_Float16)y};
            if constexpr (WIDE) {
                const h2 lo = {(_Float16)(x - (float)hi[0]), (_Float16)(y - (float)hi[1])};
                pa[i] = as_u(hi);
                pb[i] = as_u(lo);
            } else {
                const float xr = fmaf(-(float)hi[0], lo_col, x), yr = fmaf(-(float)hi[1], lo_col, y);
                pa[i] = as_u((h2){(_Float16)xr, (_Float16)yr});
            }
        }
        u4 hv[KS];
        spread<KS>(t.vh, hv);
#pragma unroll
        for (int b = 0; b < KS; ++b) {
            const u4 hw = hv[b];
            h2 off[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) off[i] = as_h2(hw[i]) * (h2){(_Float16)-72.0f, (_Float16)-72.0f};
#pragma unroll
            for (int dt = 2 * b; dt < 2 * b + 2; ++dt) {
                const uint32_t w = t.v[dt];
                const uint32_t n[4] = {w << 4, w, w >> 4, w >> 8};
                u4 va;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    va[i] = as_u(__builtin_elementwise_fma(as_h2((n[i] & 0x00f000f0u) | 0x54005400u),
                                                           as_h2(hw[i]), off[i]));
                const h8 vv = __builtin_bit_cast(h8, va);
                if constexpr (WIDE)
                    o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv, __builtin_bit_cast(h8, pb),
                                                                   o[dt], 0, 0, 0);
                o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv, __builtin_bit_cast(h8, pa), o[dt],
                                                               0, 0, 0);
            }
        }
    };
    while (s0 < p1) {
        const int s1 = s0 + A4_STEP, s2 = s1 + A4_STEP;
        if (s1 < p1) load(tb, s1, id);
        id = ids_of(s2);
        step(ta, s0);
        if (s1 >= p1) break;
        if (s2 < p1) load(ta, s2, id);
        id = ids_of(s2 + A4_STEP);
        step(tb, s1);
        s0 = s2;
    }
    // the wavefronts' states meet in LDS
    lsum += swap16_f(lsum);
    lsum += swap32_f(lsum);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
        f4 v = o[dt];
        if constexpr (!WIDE)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = ror8_add(v[i]);
        if (col < per) *(f4 *)&mo[wave][col][16 * dt + 4 * g] = v * 16.0f;
    }
    if (g == 0 && col < per) {
        mm[wave][col] = m;
        ml[wave][col] = lsum;
    }
    __syncthreads();
    if (tid < per) {
        const float M = fmaxf(fmaxf(mm[0][tid], mm[1][tid]), fmaxf(mm[2][tid], mm[3][tid]));
        float l = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mm[w][tid] - M);
            sc[tid][w] = f;
            l = fmaf(ml[w][tid], f, l);
        }
        if (ns > 1) {
            const size_t pi = ((size_t)qi * qheads + g0 * per + tid) * ns + sp;
            ws_m[pi] = M;
            ws_l[pi] = l;
        } else {
            linv[tid] = M == -INFINITY ? 0.0f : 1.0f / l;
        }
    }
    __syncthreads();
    for (int e0 = 0; e0 < per * D / 4; e0 += 256) {  // 8 lanes hold a Q8_0 block
        const int e4 = e0 + tid;
        if (e4 >= per * D / 4) break;
        const int h = e4 / (D / 4), dd = e4 % (D / 4) * 4;
        f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const f4 v = *(const f4 *)&mo[w][h][dd];
            const float f = sc[h][w];
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = fmaf(v[i], f, acc[i]);
        }
        const int head = g0 * per + h;
        if (ns > 1) {
            *(f4 *)(ws_o + (((size_t)qi * qheads + head) * ns + sp) * D + dd) = acc;
        } else {
            const float r = linv[h], y[4] = {acc[0] * r, acc[1] * r, acc[2] * r, acc[3] * r};
            const size_t off = ((size_t)qi * qheads + head) * D + dd;
#pragma unroll
            for (int i = 0; i < 4; ++i) attn[off + i] = y[i];
            if (qs) {
                uint16_t dbits;
                int sum;
                const uint32_t w = quant_block_oct(y, dbits, sum);
#pragma unroll
                for (int i = 0; i < 4; ++i) qs[off + i] = (int8_t)(w >> (8 * i));
                if ((e4 & 7) == 0) {
                    qd8[off / SI_QK] = dbits;
                    if (bsum) bsum[off / SI_QK] = (int16_t)sum;
                }
            }
        }
    }
}

// ---------------------------------------------------------------------------
// page copies: grid (pieces of a page, moves, pools); the pools' addresses and
// the moves travel in the kernel's arguments, so the call needs no upload
// ---------------------------------------------------------------------------
template <class T>
__global__ void __launch_bounds__(256) k_kv_copy(KvMoves mv, size_t page_bytes) {
    uint8_t *pool = mv.pool[blockIdx.z];
    const T *src = (const T *)(pool + (size_t)mv.src[blockIdx.y] * page_bytes);
    T *dst = (T *)(pool + (size_t)mv.dst[blockIdx.y] * page_bytes);
    const size_t n = page_bytes / sizeof(T);
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256)
        dst[i] = src[i];
}

// ---------------------------------------------------------------------------
// launchers
// ---------------------------------------------------------------------------
#define KV4_DIM(hdim, CALL)      \
    switch (hdim) {              \
        case 32: CALL(32); break; \
        case 64: CALL(64); break; \
        case 96: CALL(96); break; \
        default: CALL(128); break; \
    }

void launch_rope_kv4(const float *qkv, int ldqkv, int ntok, int qheads, int hdim, int pos0,
                     int pos_step, int max_pos, const int *ctx_dev, const float *rc,
                     const float *rs, float *q_out, const Kv4Cache &c, hipStream_t st) {
    if (ntok <= 0) return;
    const int limit = (int)min((long long)max_pos, (long long)c.max_pages << c.shift);
    const int qy = (qheads * hdim / 2 + 2 * hdim - 1) / (2 * hdim);
    const dim3 grid(kv4_units(ntok, pos0, pos_step), c.kvheads + qy);
#define CALL(DIM)                                                                               \
    SI_LAUNCH((k_kv4_append<DIM, false>), grid, dim3(2 * DIM), 0, st, qkv, ldqkv, nullptr,      \
              nullptr, qheads, ntok, pos0, pos_step, limit, ctx_dev, rc, rs, q_out, c)
    KV4_DIM(hdim, CALL)
#undef CALL
}

void launch_kv4_write(const uint16_t *k, const uint16_t *v, int ntok, int hdim, int pos0,
                      int pos_step, const int *ctx_dev, const Kv4Cache &c, hipStream_t st) {
    if (ntok <= 0) return;
    const int limit = (int)min(2147483647ll, (long long)c.max_pages << c.shift);
    const dim3 grid(kv4_units(ntok, pos0, pos_step), c.kvheads);
#define CALL(DIM)                                                                            \
    SI_LAUNCH((k_kv4_append<DIM, true>), grid, dim3(2 * DIM), 0, st, nullptr, 0, k, v, 0, ntok, \
              pos0, pos_step, limit, ctx_dev, nullptr, nullptr, nullptr, c)
    KV4_DIM(hdim, CALL)
#undef CALL
}

void launch_kv4_read(const Kv4Cache &c, int ntok, int hdim, int pos0, int pos_step,
                     const int *ctx_dev, uint16_t *k, uint16_t *v, hipStream_t st) {
    if (ntok <= 0) return;
    const int limit = (int)min(2147483647ll, (long long)c.max_pages << c.shift);
    const dim3 grid(kv4_units(ntok, pos0, pos_step), c.kvheads);
#define CALL(DIM)                                                                              \
    SI_LAUNCH((k_kv4_read<DIM>), grid, dim3(2 * DIM), 0, st, c, ntok, pos0, pos_step, limit,   \
              ctx_dev, k, v)
    KV4_DIM(hdim, CALL)
#undef CALL
}

// Chunks of the context: about 1024 workgroups, each of whole steps
static int attn_kv4_chunks(int kvheads, int nq, int max_ctx) {
    const int most = (max_ctx + A4_STEP - 1) / A4_STEP;
    const int want = (int)((1024 + (long long)kvheads * nq - 1) / ((long long)kvheads * nq));
    return max(1, min(min(most, want), 256));
}

// Whether a prompt's pages are read into fp16 rows for the prefill kernel
static bool kv4_by_rows(int nq, int ctx_step) { return ctx_step == 1 && nq > 4; }

size_t attn_kv4_workspace(int qheads, int kvheads, int hdim, int nq, int ctx_step, int max_ctx) {
    if (kv4_by_rows(nq, ctx_step)) return (size_t)max_ctx * kvheads * hdim * 2 * sizeof(uint16_t);
    const int ns = attn_kv4_chunks(kvheads, nq, max_ctx);
    return ns == 1 ? 0 : (size_t)nq * qheads * ns * (hdim + 2) * sizeof(float);
}

void launch_attention_kv4(const float *q, int nq, int qheads, int hdim, const Kv4Cache &c,
                          const int *ctx_dev, int ctx0, int ctx_step, int max_ctx, float *attn,
                          int8_t *qs, uint16_t *d, int16_t *bsum, void *ws, hipStream_t st) {
    if (nq <= 0) return;
    if (kv4_by_rows(nq, ctx_step)) {
        uint16_t *k = (uint16_t *)ws, *v = k + (size_t)max_ctx * c.kvheads * hdim;
        launch_kv4_read(c, ctx0 - 1 + nq, hdim, 0, 1, nullptr, k, v, st);
        launch_attn_prefill(q, nq, qheads, c.kvheads, hdim, ctx0 - 1, k, v, attn, qs, d, bsum, st);
        return;
    }
    const int ns = attn_kv4_chunks(c.kvheads, nq, max_ctx);
    const int chunk = ((max_ctx + ns - 1) / ns + A4_STEP - 1) / A4_STEP * A4_STEP;
    const AttnParts pt(ws, (size_t)nq * qheads * ns, hdim);
    const dim3 grid(ns, c.kvheads, nq);
    const bool wide = qheads / c.kvheads > 8, page16 = c.shift == 4;
#define CALL2(DIM, W, P)                                                                            SI_LAUNCH((k_attn_kv4<DIM, W, P>), grid, dim3(256), 0, st, q, qheads, c, ctx_dev, ctx0,                   ctx_step, max_ctx, chunk, softmax_scale2(hdim), pt.m, pt.l, pt.o, attn, qs, d, bsum)
#define CALL(DIM)                                              if (wide && page16) CALL2(DIM, true, true);                else if (wide) CALL2(DIM, true, false);                    else if (page16) CALL2(DIM, false, true);                  else CALL2(DIM, false, false)
    KV4_DIM(hdim, CALL)
#undef CALL
#undef CALL2
    if (ns > 1) launch_attn_combine(nq, qheads, hdim, ns, ws, attn, qs, d, bsum, st);
}

void launch_kv_copy(const KvMoves &mv, int npools, int nmoves, size_t page_bytes, bool wide,
                    hipStream_t st) {
    const size_t unit = wide ? 16 : 1;
    const size_t want = (page_bytes / unit + 256 * 4 - 1) / (256 * 4);
    const dim3 grid((unsigned)min(want, (size_t)64), nmoves, npools);
    if (wide) SI_LAUNCH(k_kv_copy<uint4>, grid, dim3(256), 0, st, mv, page_bytes);
    else SI_LAUNCH(k_kv_copy<uint8_t>, grid, dim3(256), 0, st, mv, page_bytes);
}
}  // namespace si
