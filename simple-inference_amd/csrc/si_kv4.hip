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
// pos0).  Tokens t0 + j sit at base + j for j in [lo, hi).  A device context past
// `limit` is skipped, or taken as limit (clamp).
struct Kv4Unit {
    int seq, base, t0, lo, hi;
    __device__ __forceinline__ Kv4Unit(int x, int ntok, int pos0, int pos_step,
                                       const int *ctx_dev, int limit, bool clamp = false) {
        if (pos_step) {
            seq = 0;
            base = (pos0 & ~7) + 8 * x;
            t0 = base - pos0;
            lo = max(-t0, 0);
            hi = min(min(ntok - t0, limit - base), 8);
        } else {
            int ctx = ctx_dev ? ctx_dev[x] : pos0 + 1;
            if (clamp) ctx = min(ctx, limit);
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
// A thread per position and octet of dims, D for K and D for V, a block's four
// octets in a quad of lanes.  V's nibbles pass through LDS to a thread per dim,
// whose dword holds the unit's 8 positions (one that is not written whole keeps
// its other nibbles).  (V by a thread per dim with all 8 positions took 8
// reductions over 32 lanes one after another: 5000 fp16 rows of 2 heads of 128
// 7.0 us, 5.0 so.)
// HALF_IN: the rows are fp16 cache rows (kin, vin), copied in without RoPE.
// Many rows are bound by memory: 1999 rows of 28/4 heads of 128, 68 MB with q in
// and out, 13.8 us; 77 MB move, as each XCD reads the tables for itself, at 5.6 TB/s
// (k_kv_copy reaches 5.9).  Few by their launch and one chain of loads, reduction and
// store: 64 rows 4.3 us, 1 row 3.4, 5000 fp16 rows of 2 heads of 128 (6.6 MB) 5.0.
// ---------------------------------------------------------------------------
// 8 floats, 16 bytes a load where the call's buffers allow it
__device__ __forceinline__ void load8(const float *p, bool wide, float (&v)[8]) {
    if (wide) {
        const float4 a = *(const float4 *)p, b = *(const float4 *)(p + 4);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
        v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = p[e];
    }
}

template <int D, bool HALF_IN>
__global__ void __launch_bounds__(2 * D) k_kv4_append(
    const float *__restrict__ qkv, int ldqkv, const uint16_t *__restrict__ kin,
    const uint16_t *__restrict__ vin, int qheads, int ntok, int pos0, int pos_step, int limit,
    const int *__restrict__ ctx_dev, const float *__restrict__ rc, const float *__restrict__ rs,
    float *__restrict__ q_out, bool wide, bool clamp, Kv4Cache c) {
    constexpr int HALF = D / 2;
    const Kv4Unit un((int)blockIdx.x, ntok, pos0, pos_step, ctx_dev, limit, clamp);
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
    __shared__ __attribute__((aligned(8))) uint8_t vn[D][8];  // V's nibbles [dim][position]
    const bool is_k = tid < D;
    const int t = is_k ? tid : tid - D, j = t / (D / 8), o = t % (D / 8);
    const int pos = un.base + j, i = in_page + j;
    const bool live = j >= un.lo && j < un.hi;
    float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (live) {
        if constexpr (HALF_IN) {
            const uint4 w = *(const uint4 *)((is_k ? kin : vin) + (size_t)(un.t0 + j) * kvd +
                                             g * D + 8 * o);
            const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = h2f_fast((uint16_t)(v[e / 2] >> (16 * (e & 1))));
        } else {
            const float *row = qkv + (size_t)(un.t0 + j) * ldqkv + qd + g * D;
            if (is_k) {
                const int i0 = 8 * o < HALF ? 8 * o : 8 * o - HALF;  // (8 divides HALF)
                float a[8], b[8], cs[8], sn[8];
                load8(row + i0, wide, a);
                load8(row + i0 + HALF, wide, b);
                load8(rc + (size_t)pos * HALF + i0, wide, cs);
                load8(rs + (size_t)pos * HALF + i0, wide, sn);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    x[e] = 8 * o < HALF ? __fsub_rn(__fmul_rn(a[e], cs[e]), __fmul_rn(b[e], sn[e]))
                                        : __fadd_rn(__fmul_rn(b[e], cs[e]), __fmul_rn(a[e], sn[e]));
            } else {
                load8(row + kvd + 8 * o, wide, x);
            }
        }
    }
    uint32_t key = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        x[e] = x[e] == x[e] ? x[e] : 0.0f;
        key = max(key, kv4_key(x[e]));
    }
    key = max(key, (uint32_t)dpp_i<DPP_XOR1>((int)key));
    key = max(key, (uint32_t)dpp_i<DPP_XOR2>((int)key));
    const uint16_t h = kv4_scale_of(key);
    const Kv4Scale sc(h);
    uint8_t *page = (is_k ? c.k : c.v) + at;
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t n = sc.nibble(x[e]);
        w |= n << (4 * e);
        if (!is_k) vn[8 * o + e][j] = (uint8_t)n;
    }
    if (live) {
        if (is_k) *(uint32_t *)(page + kv4_k_dword(D, i, o)) = w;
        if ((o & 3) == 0) *(uint16_t *)(page + kv4_scale(D, page_size, i, o >> 2)) = h;
    }
    __syncthreads();
    if (!is_k) {  // a thread per dim: bytes n0 .. n7 to one dword
        const uint2 n = *(const uint2 *)vn[t];
        const uint32_t lo = n.x | n.x >> 4, hi = n.y | n.y >> 4;  // n0 + n1 * 16 in byte 0, ..
        const uint32_t v = __builtin_amdgcn_perm(hi, lo, 0x06040200u);
        const uint32_t some = un.hi - un.lo == 8
                                  ? 0xffffffffu
                                  : ((1u << (4 * (un.hi - un.lo))) - 1) << (4 * un.lo);
        uint32_t *dst = (uint32_t *)(page + kv4_v_dword(D, in_page >> 3, t));
        *dst = some == 0xffffffffu ? v : (*dst & ~some) | (v & some);
    }
}

// ---------------------------------------------------------------------------
// rows back as fp16, exactly: the same units and threads.  A launch and one chain
// of loads (page id, nibbles and scale): 1 row 2.3 us, 1999 rows of 4 heads of 128
// (5.2 MB) 4.2, 5000 of 2 (6.6 MB) 4.2.
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
    // V's dwords pass through LDS to a thread per position and octet, like K's
    __shared__ __attribute__((aligned(16))) uint32_t vw[D];
    const bool is_k = tid < D;
    const int t = is_k ? tid : tid - D, j = t / (D / 8), o = t % (D / 8), i = in_page + j;
    const uint8_t *page = (is_k ? c.k : c.v) + at;
    if (!is_k) vw[t] = *(const uint32_t *)(page + kv4_v_dword(D, in_page >> 3, t));
    __syncthreads();
    if (j < un.lo || j >= un.hi) return;
    const uint16_t h = *(const uint16_t *)(page + kv4_scale(D, page_size, i, o >> 2));
    const float d = h2f_fast(h) * 16.0f;
    uint32_t w = 0;
    if (is_k) {
        w = *(const uint32_t *)(page + kv4_k_dword(D, i, o));
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) w |= (vw[8 * o + e] >> (4 * j) & 15u) << (4 * e);
    }
    uint32_t y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const _Float16 a = (_Float16)((float)((int)(w >> (8 * e) & 15) - 8) * d);
        const _Float16 b = (_Float16)((float)((int)(w >> (8 * e + 4) & 15) - 8) * d);
        y[e] = __builtin_bit_cast(uint16_t, a) | (uint32_t)__builtin_bit_cast(uint16_t, b) << 16;
    }
    *(uint4 *)((is_k ? kout : vout) + (size_t)(un.t0 + j) * kvd + g * D + 8 * o) =
        make_uint4(y[0], y[1], y[2], y[3]);
}

// ---------------------------------------------------------------------------
// attention over the pages: a workgroup per (KV head, query, context chunk), or per
// 16 rows (query, head) of a prompt, whose NW wavefronts take every NW-th group of
// 32 positions.  Per group
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
// fp16 roundings of q the result was off by up to 2.7e-5).  With at most 8 heads a
// KV head both halves share one product: columns 0-7 carry hi, 8-15 lo, and their
// results are added across (WIDE: 9 to 16 heads, two products).
//
// A column's running maximum is moved only when a score of its own passes it by 2^4,
// in a branch that the wavefront takes together: no head's bits depend on the other
// heads'.  A weight w against it, up to 2^4, goes in as w 2^11 (fp16 holds 2^16),
// its lo half 2^11 higher still and in sums of its own (the lo columns', or WIDE's
// second accumulators), so that the pair has 22 bits down to w = 2^-25 and an error of
// at most 2^-47 below: a position with all the weight and a zero V row leaves the
// others their bits up to 20 nats under it.  (In the same units and sums as hi, lo
// was an fp16 subnormal from w = 2^-3 down and weights below 2^-25 were 0: 1.6e-5 of
// the result 10 nats under such a position, all of a wavefront's at 18.)
//
// What bounds it: a step of 32 positions is about 240 vector operations and 17 matrix
// instructions (two products: 270 and 34), which hardly overlap, 0.7 us of a SIMD at
// 128 dims, about as long as its 4.6 KB take to arrive.  64 queries x 4096 of 28/4 heads
// of 128, 153 MB: 32.6 us (4.7 TB/s; a plain read takes 28), vector issue busy half of it
// and the matrix cores an eighth.  Fewer bytes leave 5 us of launch, page id, first
// group, last step and the wavefronts' meeting, and the merge of chunks: 48 x 200-4096
// (62 MB) 21 + 4 us, 2 queries of 12/2 heads over 60000-131072 (65 MB) 19 + 4, one query
// of 14/2 heads of 64 over 1024 (no merge) 7.9.
// ---------------------------------------------------------------------------
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int A4_GROUP = 32;  // positions of a wavefront's step
constexpr float A4_SLACK = 4.0f;  // log2 of the largest weight
constexpr float A4_UP = 11.0f;    // log2 of a weight's unit in hi
constexpr float A4_LO = 2048.0f;  // and of lo's in hi's

__device__ __forceinline__ float ror8_add(float v) { return v + dpp_f<DPP_ROR8>(v); }

// Where a wavefront reads: one page's part of a KV head, as a buffer descriptor
// (the group's place in it is the load's scalar offset, so a step computes no
// addresses in vector registers, and nothing past the page is touched), or, for
// pages of half a group, the lane's own address.
// ONCE: no other workgroup reads the bytes soon (every query but a prompt's), so they
// are loaded past the caches, which the next layers' pages then find as they were: 64
// queries x 4096 of 28/4 heads of 128 from memory 37.8 -> 37.5 us, 200 x 2000 59.3 -> 56.2,
// 8 x 4096 14.3 -> 14.5, 128 x 4000 of 14/2 of 64 24.7 -> 23.2 (2.5 GB of other pages
// between; the same pages again and again from the 256 MB cache 31.3 -> 34.0, 50.2 -> 55.0,
// 12.7 -> 13.1, 21.4 -> 22.4).  A prompt, whose blocks of rows share them, 85.5 -> 88.7.
struct Kv4InPage {
    __amdgpu_buffer_rsrc_t r;
    int at;
    template <int N, bool ONCE>
    __device__ __forceinline__ void load(int off, uint32_t *w) const {
        constexpr int AUX = ONCE ? 2 : 0;  // nt
        if constexpr (N == 1) {
            w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, off, at, AUX);
        } else if constexpr (N == 2) {
            const auto t = __builtin_amdgcn_raw_buffer_load_b64(r, off, at, AUX);
            w[0] = t[0], w[1] = t[1];
        } else if constexpr (N == 3) {
            const auto t = __builtin_amdgcn_raw_buffer_load_b96(r, off, at, AUX);
            w[0] = t[0], w[1] = t[1], w[2] = t[2];
        } else {
            const auto t = __builtin_amdgcn_raw_buffer_load_b128(r, off, at, AUX);
            w[0] = t[0], w[1] = t[1], w[2] = t[2], w[3] = t[3];
        }
    }
};
struct Kv4InHalf {
    const uint8_t *p;
    template <int N, bool ONCE>
    __device__ __forceinline__ void load(int off, uint32_t *w) const {
        // (three dwords as such: rows of 12 bytes are 4-byte aligned)
        typedef uint32_t vec __attribute__((ext_vector_type(N == 3 ? 1 : N)));
        constexpr int PER = N == 3 ? 1 : N;
#pragma unroll
        for (int e = 0; e < N; e += PER) {
            const vec *a = (const vec *)(p + off + 4 * e);
            vec t;
            if constexpr (ONCE) t = __builtin_nontemporal_load(a);
            else t = *a;
#pragma unroll
            for (int i = 0; i < PER; ++i) w[e + i] = t[i];
        }
    }
};

// What a wavefront reads of a group: lane (col, g)'s K nibbles of both tiles, V
// nibbles, and dword col of the D / 8 dwords that hold the scales of positions
// 8 g .. 8 g + 7: all 16 lanes of a row need them all, and read them from the
// wavefront's own room in LDS (as DPP broadcasts they were 48 of a step's 275
// vector operations, what bounds the kernel; loaded by every lane, 32 registers
// and 8 of the 14 loads).
template <int D, bool ONCE>
struct Kv4Group {
    static constexpr int KS = D / 32, DT = D / 16;
    uint32_t k[2][KS], v[DT], kh, vh;
    // ku, vu: the places of the K row's and the V positions' unit
    template <class P>
    __device__ __forceinline__ void load(const P &kk, const P &ks, const P &vv, const P &vs,
                                         int ku, int vu, int lane) {
        const int r = lane & 15, g = lane >> 4;
        const int so = vu * KS * 16 + min(r, 4 * KS - 1) * 4;
        ks.template load<1, false>(so, &kh);  // (a line holds several groups')
        vs.template load<1, false>(so, &vh);
#pragma unroll
        for (int t = 0; t < 2; ++t)
            kk.template load<KS, ONCE>(ku * 4 * D + t * 2 * D + g * (D / 2) + (r & 3) * (D / 8),
                                       k[t]);
        constexpr int FULL = D / 64;
#pragma unroll
        for (int f = 0; f < FULL; ++f)
            vv.template load<4, ONCE>(vu * 4 * D + f * 256 + r * 16, v + 4 * f);
        if constexpr (DT % 4)
            vv.template load<2, ONCE>(vu * 4 * D + FULL * 256 + r * 8, v + 4 * FULL);
    }
};

__device__ __forceinline__ h2 as_h2(uint32_t u) { return __builtin_bit_cast(h2, u); }
__device__ __forceinline__ uint32_t as_u(h2 h) { return __builtin_bit_cast(uint32_t, h); }
__device__ __forceinline__ h8 to_h8(const float (&x)[8]) {
    h8 y;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = (_Float16)x[e];
    return y;
}

// An oct's 32 outputs, 4 a lane (lane l8 at off), and their Q8_0; row qi of qd
// values in the operand-tiled copy.
__device__ __forceinline__ void kv4_store(const float (&y)[4], size_t off, int l8, float *attn,
                                          int8_t *qs, uint16_t *d, int16_t *bsum, int8_t *tq,
                                          uint16_t *td, int qd, int qi) {
#pragma unroll
    for (int i = 0; i < 4; ++i) attn[off + i] = y[i];
    if (!qs) return;
    uint16_t dbits;
    int sum;
    const uint32_t w = quant_block_oct(y, dbits, sum);
#pragma unroll
    for (int i = 0; i < 4; ++i) qs[off + i] = (int8_t)(w >> (8 * i));
    const size_t pb = (size_t)(qi >> 5) * (qd / SI_QK) + off % qd / SI_QK;
    if (tq) *(uint32_t *)(tq + q8_tiled_byte(pb, qi & 31, 4 * l8)) = w;
    if (l8 == 0) {
        d[off / SI_QK] = dbits;
        if (bsum) bsum[off / SI_QK] = (int16_t)sum;
        if (tq) td[pb * 32 + (qi & 31)] = dbits;
    }
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ float uniform(float v) { return u2f((uint32_t)uniform((int)f2u(v))); }
// inclusive sum over the wavefront's lanes before this one and its own
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15, 31
    return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
}

// Which chunk of which query a workgroup takes.
struct A4Item {
    int qi, sp, ctx, chunk, parts;  // parts: chunks of the query; ctx 0: nothing to do
};
// Contexts on the device: item w of the list of all queries' chunks, in order.
// The chunk makes about `slots` of them in all, what the GPU holds at once, by
// sum of ctx_i / chunk + half a chunk a query for the last ones (never over slots /
// kvheads + nq, the launch), and the longest context's chunks equal; at most ns a
// query.  (A grid of query x chunk instead, each workgroup past its context
// leaving at once, kept the slots busy with those: 48 x 200-4096 24.8 us
// against 21.3.)
template <int step>
__device__ __forceinline__ A4Item a4_item(int w, const int *ctx_dev, int nq, int kvheads, int ns,
                                          int max_ctx, int slots) {
    const int lane = threadIdx.x & 63;
    int most = 0, live = 0;
    float total = 0.0f;
    const int first = lane < nq ? max(min(ctx_dev[lane], max_ctx), 0) : 0;
    for (int i = lane; i < nq; i += 64) {
        const int n = i < 64 ? first : max(min(ctx_dev[i], max_ctx), 0);
        most = max(most, n);
        total += (float)n;
        live += n > 0;
    }
    most = max(uniform(wave_max_i(most)), 1);
    total = uniform(wave_sum(total));
    const float n = uniform(wave_sum((float)live));
    const float share = total / fmaxf((float)slots / (float)kvheads - 0.5f * n, 1.0f);
    const int k = min((int)((float)most / fmaxf(share, (float)step)), ns);
    auto steps_of = [&](int k) { return ((most + k - 1) / k + step - 1) / step; };
    auto parts_of = [](int ctx, int steps) {
        return ((ctx + step - 1) / step + steps - 1) / steps;
    };
    int steps = steps_of(max(k, 1));
    if (k < ns) {  // one chunk more where that still fits (equal contexts)
        const int more = steps_of(k + 1);
        int count = 0;
        for (int i = lane; i < nq; i += 64)
            count += parts_of(i < 64 ? first : max(min(ctx_dev[i], max_ctx), 0), more);
        if (uniform(wave_sum((float)count)) * (float)kvheads <= (float)slots) steps = more;
    }
    A4Item it = {0, 0, 0, steps * step, 0};
    for (int i0 = 0; i0 < nq; i0 += 64) {
        const int i = i0 + lane;
        const int c = i >= nq ? 0 : i0 == 0 ? first : max(min(ctx_dev[i], max_ctx), 0);
        const int parts = parts_of(c, steps);
        const int upto = wave_scan(parts);
        const unsigned long long past = __ballot(upto > w);
        if (past) {
            const int l = uniform((int)__builtin_ctzll(past));
            it.qi = i0 + l;
            it.ctx = __builtin_amdgcn_readlane(c, l);
            it.parts = __builtin_amdgcn_readlane(parts, l);
            it.sp = w - (__builtin_amdgcn_readlane(upto, l) - it.parts);
            break;
        }
        w -= __builtin_amdgcn_readlane(upto, 63);
    }
    return it;
}

// What a workgroup's columns are: one query's heads, up to 8 in hi and lo columns, or
// up to 16 in two products; or 16 rows (query, head) of a prompt, whose contexts
// end query by query.
enum A4Mode { A4_NARROW, A4_WIDE, A4_ROWS };

template <int D, int MODE, bool PAGE16, int NW>
__global__ void __launch_bounds__(64 * NW, 3) k_attn_kv4(
    const float *__restrict__ q, int qheads, Kv4Cache c, const int *__restrict__ ctx_dev, int ctx0,
    int ctx_step, int nq, int max_ctx, int ns, int chunk, int slots, float scale2,
    int *__restrict__ parts, float *__restrict__ ws_u, float *__restrict__ ws_m,
    float *__restrict__ ws_l, float *__restrict__ ws_o, float *__restrict__ attn,
    int8_t *__restrict__ qs, uint16_t *__restrict__ qd8, int16_t *__restrict__ bsum,
    int8_t *__restrict__ tq, uint16_t *__restrict__ td) {
    constexpr bool WIDE = MODE != A4_NARROW, ROWS = MODE == A4_ROWS;
    typedef Kv4Group<D, !ROWS> Group;
    constexpr int KS = D / 32, DT = D / 16, COLS = WIDE ? 16 : 8, STEP = NW * A4_GROUP;
    __shared__ __attribute__((aligned(16))) float mo[4][COLS][D];
    __shared__ __attribute__((aligned(16))) u4 qop[(WIDE ? 2 : 1) * KS * 64];  // hi (, lo)
    __shared__ __attribute__((aligned(16))) f4 qc[(WIDE ? 2 : 1) * KS * 64];
    __shared__ __attribute__((aligned(16))) uint32_t scales[NW][3][64];  // K's, V's, V's * -72
    __shared__ float mm[NW][COLS], ml[NW][COLS], sc[COLS][NW], linv[COLS], units[COLS];
    const int g0 = blockIdx.x, per = qheads / c.kvheads;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = uniform(tid >> 6);
    const int col = lane & 15, g = lane >> 4;
    // rows of this workgroup, the first of all its KV head's; their heads in q and
    // the outputs
    const int row0 = ROWS ? 16 * (int)blockIdx.y : 0;
    const int rows = ROWS ? min(16, nq * per - row0) : per;
    A4Item it;
    if (!ROWS && parts) {
        it = a4_item<STEP>(blockIdx.y, ctx_dev, nq, c.kvheads, ns, max_ctx, slots);
        if (it.ctx == 0) return;  // past the list
        if (g0 == 0 && it.sp == 0 && tid == 0) parts[it.qi] = it.parts;
    } else {
        it.qi = ROWS ? (row0 + rows - 1) / per : blockIdx.y;  // (the last one)
        it.sp = blockIdx.z;
        it.ctx = min(ctx_dev ? ctx_dev[it.qi] : ctx0 + it.qi * ctx_step, max_ctx);
        it.chunk = chunk;
        it.parts = ns;
    }
    const int qi = uniform(it.qi), sp = uniform(it.sp), seq = ctx_step ? 0 : qi;
    const int p0 = uniform(sp * it.chunk), p1 = uniform(min(it.ctx, p0 + it.chunk));
    auto head_of = [&](int r) {
        if constexpr (ROWS) {
            const int qr = (row0 + r) / per;
            return (size_t)qr * qheads + g0 * per + (row0 + r - qr * per);
        } else {
            return (size_t)qi * qheads + g0 * per + r;
        }
    };
    // positions that the lane's column sees end at `end`, every column's at `all` or past it
    const int end = ROWS ? min(ctx0 + (row0 + min(col, rows - 1)) / per, p1) : p1;
    const int all = ROWS ? uniform(min(ctx0 + row0 / per, p1)) : p1;
    // groups of this wavefront: s0 = p0 + 32 wave, + STEP, ...
    const int page_size = 1 << c.shift, nib = page_size * (D / 2);
    const size_t hb = (size_t)kv4_head_bytes(D, page_size);
    // (constant memory: scalar loads, which the vector loads' order does not wait for)
    typedef const __attribute__((address_space(4))) int *const_ints;
    const const_ints pages = (const_ints)(uintptr_t)(c.pages + (size_t)seq * c.max_pages);
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
    auto load = [&](Group &t, int s0, Ids id) {
        const size_t a = head_at(id.a);
        if constexpr (PAGE16) {
            // two pages a group: units 0, 1 and 2, 3
            const size_t b = head_at(id.b);
            const size_t ka = (lane & 8) ? b : a, va = (lane & 32) ? b : a;
            t.load(Kv4InHalf{c.k + ka}, Kv4InHalf{c.k + va + nib}, Kv4InHalf{c.v + va},
                   Kv4InHalf{c.v + va + nib}, (lane >> 2) & 1, g & 1, lane);
        } else {
            const int u = (s0 & (page_size - 1)) >> 3, sc = nib + u * KS * 16;
            const auto rk = buf_rsrc(c.k + a, (uint32_t)hb), rv = buf_rsrc(c.v + a, (uint32_t)hb);
            t.load(Kv4InPage{rk, u * 4 * D}, Kv4InPage{rk, sc}, Kv4InPage{rv, u * 4 * D},
                   Kv4InPage{rv, sc}, (lane >> 2) & 3, g, lane);
        }
    };
    int s0 = p0 + A4_GROUP * wave;
    Group ta, tb;
    {
        const Ids ia = ids_of(s0), ib = ids_of(s0 + STEP);
        if (s0 < p1) load(ta, s0, ia);
        if (s0 + STEP < p1) load(tb, s0 + STEP, ib);
    }
    Ids id = ids_of(s0 + 2 * STEP);

    // q of the lane's column as the B operand, dims 32 b + 8 g + (0, 4, 1, 5, 2, 6,
    // 3, 7), the odd ones over 16: integers hi and lo, q = (hi + lo 2^-12) 2^(ex - 10)
    // (lo 2^-12 is the operand: a 12-bit integer over 2^16 is an fp16 value).
    // Wavefront b makes block b for all of them (each making all took 370
    // operations of a wavefront's 250 a step); the operands and -8 sum q stay in LDS
    // and are read again in each step (kept in registers they are 32 of them, the
    // difference between three wavefronts a SIMD and two).
    float fac;
    const bool lo_half = !WIDE && col >= 8;
    const float lo_col = lo_half ? A4_LO : 0.0f, lo_mul = lo_half ? A4_LO : 1.0f;
    {
        float *qmax = &mo[0][0][0];  // [KS][64]
        const int hc = WIDE ? col : col & 7;
        float x[8];
        if (wave < KS) {
            const float *row = q + head_of(min(hc, rows - 1)) * D + 32 * wave + 8 * g;
            float big = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = row[e];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = hc < rows ? x[e] : 0.0f;
                big = fmaxf(big, fabsf(x[e]));
            }
            qmax[wave * 64 + lane] = big;
        }
        __syncthreads();
        float big = 0.0f;
#pragma unroll
        for (int b = 0; b < KS; ++b) big = fmaxf(big, qmax[b * 64 + lane]);
        big = fmaxf(big, swap16_f(big));
        big = fmaxf(big, swap32_f(big));
        const int ex = big == 0.0f ? 0 : (int)(f2u(big) >> 23) - 127;
        // the scores' units: 2^24 of the subnormals, 16 of the scale, q's (finite for
        // the largest q too, whose weights are then 0 or 1 either way)
        fac = fminf(__builtin_amdgcn_ldexpf(scale2, 28 + ex - 10), 0x1.fffffep127f);
        if (wave < KS) {
            float hi[8], lo[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int dim = (e >> 1) + (e & 1) * 4;
                const float y = __builtin_amdgcn_ldexpf(x[dim], 10 - ex);
                const float odd = (dim & 1) ? 0.0625f : 1.0f;
                hi[e] = rintf(y) * odd;
                lo[e] = rintf((y - rintf(y)) * 4096.0f) * (odd * 0x1p-12f);
                if (!WIDE) hi[e] = lo_half ? lo[e] : hi[e];
            }
            qop[wave * 64 + lane] = __builtin_bit_cast(u4, to_h8(hi));
            if constexpr (WIDE) qop[(KS + wave) * 64 + lane] = __builtin_bit_cast(u4, to_h8(lo));
        }
        const u4 eight = {0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u};  // -8 in K's units
        if (wave < KS) {
#pragma unroll
            for (int w = 0; w < (WIDE ? 2 : 1); ++w) {
                const h8 x8 = __builtin_bit_cast(h8, qop[(w * KS + wave) * 64 + lane]);
                qc[(w * KS + wave) * 64 + lane] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                    __builtin_bit_cast(h8, eight), x8, (f4){0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
            }
        }
        __syncthreads();
    }
    // The running maximum m stays in the scores' raw units (fac makes them powers of
    // two): weights are 2^((s - m) fac), whose error goes with the difference, not
    // with the scores, and a score passes m by a difference too (m + over would round
    // up to 2 over where that is about m's last place).  The sums of the weights are
    // one more product's rows (ones . P), like the outputs in hi and lo.
    const float over = A4_SLACK * __builtin_amdgcn_rcpf(fac);
    // ref: m, or 0 while a column has seen no position.
    float m = -INFINITY, ref = 0.0f;
    constexpr int LO = WIDE ? DT : 0;  // WIDE: the lo halves' sums
    f4 o[DT], ol = {0.0f, 0.0f, 0.0f, 0.0f}, o2[LO + 1], ol2 = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int dt = 0; dt < LO; ++dt) o2[dt] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
    // constants held in registers, so that (n & mask) | magic is one operation
    uint32_t mask = 0x00f000f0u, magic = 0x54005400u;
    asm("" : "+s"(mask));
    asm("" : "+v"(magic));

    auto step = [&](Group &t, int s) {
        float p[2][4];
        // lane (col, g)'s dword to [g][col]; a wavefront's LDS operations keep their
        // order, the compiler is to keep it too (and to read q here, not before the
        // loop)
        uint32_t (*const sl)[64] = scales[wave];
        const bool tail = s + A4_GROUP > all;  // wavefront-uniform: positions past an end
        if (s + A4_GROUP > p1) {
            // their V scales may be anything: 0 (weight 0 * NaN would stay); dword col
            // holds positions 8 g + col % 4 and 4 further
            const int at = s + 8 * g + (col & 3);
            t.vh &= (at < p1 ? 0xffffu : 0u) | (at + 4 < p1 ? 0xffff0000u : 0u);
        }
        asm volatile("" ::: "memory");
        sl[0][lane] = t.kh;
        sl[1][lane] = t.vh;
        sl[2][lane] = as_u(as_h2(t.vh) * (h2){(_Float16)-72.0f, (_Float16)-72.0f});
        asm volatile("" ::: "memory");
        f4 acc[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
        for (int b = 0; b < KS; ++b) {
            // (q read as it is needed, or the registers are not three wavefronts' a SIMD)
            if constexpr (WIDE && D == 128) asm volatile("" ::: "memory");
            const h8 qa = __builtin_bit_cast(h8, qop[b * 64 + lane]);
            const f4 c8 = qc[b * 64 + lane];
            f4 d[2];
#pragma unroll
            for (int tl = 0; tl < 2; ++tl) {
                const uint32_t w = t.k[tl][b], w8 = w >> 8;
                const u4 a = {w & 0x000f000fu, w & 0x00f000f0u, w8 & 0x000f000fu, w8 & 0x00f000f0u};
                const h8 ka = __builtin_bit_cast(h8, a);
                d[tl] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qa, c8, 0, 0, 0);
                if constexpr (WIDE)
                    d[tl] += __builtin_amdgcn_mfma_f32_16x16x32_f16(
                        ka, __builtin_bit_cast(h8, qop[(KS + b) * 64 + lane]),
                        qc[(KS + b) * 64 + lane], 0, 0, 0);
            }
            const u4 hk = *(const u4 *)&sl[0][16 * g + 4 * b];
#pragma unroll
            for (int tl = 0; tl < 2; ++tl)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    acc[tl][i] = fmaf((float)as_h2(hk[i])[tl], d[tl][i], acc[tl][i]);
        }
#pragma unroll
        for (int tl = 0; tl < 2; ++tl)
#pragma unroll
            for (int i = 0; i < 4; ++i) p[tl][i] = WIDE ? acc[tl][i] : ror8_add(acc[tl][i]);
        if (tail) {
            int left = end - s - 8 * g;
            asm volatile("" : "+v"(left));  // (a branch, not selects in every step)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                p[0][i] = i < left ? p[0][i] : -INFINITY;
                p[1][i] = 4 + i < left ? p[1][i] : -INFINITY;
            }
        }
        float mx = fmaxf(fmaxf(fmaxf(p[0][0], p[0][1]), fmaxf(p[0][2], p[0][3])),
                         fmaxf(fmaxf(p[1][0], p[1][1]), fmaxf(p[1][2], p[1][3])));
        if (__ballot(mx - m > over)) {
            mx = fmaxf(mx, swap16_f(mx));
            mx = fmaxf(mx, swap32_f(mx));
            const float mn = mx - m > over ? mx : m;  // the column's own, whatever the others do
            const float al = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mn) * fac);
            m = mn;
            ref = mn == -INFINITY ? 0.0f : mn;
            ol *= al;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[dt] *= al;
            if constexpr (WIDE) ol2 *= al;
#pragma unroll
            for (int dt = 0; dt < LO; ++dt) o2[dt] *= al;
        }
        u4 pa, pb;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f2 x = {__builtin_amdgcn_exp2f(fmaf(p[0][i] - ref, fac, A4_UP)),
                          __builtin_amdgcn_exp2f(fmaf(p[1][i] - ref, fac, A4_UP))};
            const h2 hi = __builtin_convertvector(x, h2);
            if constexpr (WIDE) {
                pa[i] = as_u(hi);
                pb[i] = as_u((h2){(_Float16)fmaf(-(float)hi[0], A4_LO, x[0] * A4_LO),
                                  (_Float16)fmaf(-(float)hi[1], A4_LO, x[1] * A4_LO)});
            } else {
                pa[i] = as_u((h2){(_Float16)fmaf(-(float)hi[0], lo_col, x[0] * lo_mul),
                                  (_Float16)fmaf(-(float)hi[1], lo_col, x[1] * lo_mul)});
            }
        }
        const h8 ph = __builtin_bit_cast(h8, pa), pl = __builtin_bit_cast(h8, pb);
        const u4 ones = {0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
        const h8 one = __builtin_bit_cast(h8, ones);
        if constexpr (WIDE) ol2 = __builtin_amdgcn_mfma_f32_16x16x32_f16(one, pl, ol2, 0, 0, 0);
        ol = __builtin_amdgcn_mfma_f32_16x16x32_f16(one, ph, ol, 0, 0, 0);
#pragma unroll
        for (int b = 0; b < KS; ++b) {
            const u4 hv = *(const u4 *)&sl[1][16 * g + 4 * b];
            const u4 off = *(const u4 *)&sl[2][16 * g + 4 * b];
#pragma unroll
            for (int dt = 2 * b; dt < 2 * b + 2; ++dt) {
                const uint32_t w = t.v[dt];
                const uint32_t n[4] = {w << 4, w, w >> 4, w >> 8};
                u4 va;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    va[i] = as_u(__builtin_elementwise_fma(as_h2((n[i] & mask) | magic),
                                                           as_h2(hv[i]), as_h2(off[i])));
                const h8 vv = __builtin_bit_cast(h8, va);
                if constexpr (WIDE)
                    o2[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv, pl, o2[dt], 0, 0, 0);
                o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv, ph, o[dt], 0, 0, 0);
            }
        }
    };
    // (two whole steps a turn: with an exit between them the sums moved to other
    // registers and back each turn, which were then a third more)
    while (s0 + STEP < p1) {
        step(ta, s0);
        s0 += STEP;
        if (s0 + STEP < p1) load(ta, s0 + STEP, id);
        id = ids_of(s0 + 2 * STEP);
        step(tb, s0);
        s0 += STEP;
        if (s0 + STEP < p1) load(tb, s0 + STEP, id);
        id = ids_of(s0 + 2 * STEP);
    }
    if (s0 < p1) step(ta, s0);
    // The wavefronts' states meet in LDS: maxima and sums, then the outputs, four
    // wavefronts at a time, added by a thread per four dims in wavefront order.
    const float lo_unit = lo_half ? 1.0f / A4_LO : 1.0f;
    const float lsum = WIDE ? fmaf(ol2[0], 1.0f / A4_LO, ol[0]) : ror8_add(ol[0] * lo_unit);
    if (lsum != lsum) m = 0.0f;  // no score of a NaN query passes a limit: not an empty state
    if (g == 0 && col < rows) {
        mm[wave][col] = m;
        ml[wave][col] = lsum;
        if (wave == 0) units[col] = fac;
    }
    const bool whole = it.parts == 1;  // the query's only chunk
    __syncthreads();
    if (tid < rows) {
        float M = mm[0][tid], l = 0.0f;
#pragma unroll
        for (int w = 1; w < NW; ++w) M = fmaxf(M, mm[w][tid]);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float f = mm[w][tid] == -INFINITY  // no position (M may be none too)
                                ? 0.0f
                                : __builtin_amdgcn_exp2f((mm[w][tid] - M) * units[tid]);
            sc[tid][w] = f;
            l = fmaf(ml[w][tid], f, l);
        }
        if (whole) {
            linv[tid] = M == -INFINITY ? 0.0f : 1.0f / l;
        } else {
            const size_t head = head_of(tid), pi = head * ns + sp;
            ws_m[pi] = M;
            ws_l[pi] = l;
            if (sp == 0) ws_u[head] = units[tid];
        }
    }
    constexpr int SLOTS = (COLS * D / 4 + 64 * NW - 1) / (64 * NW);  // of a thread
    f4 acc[SLOTS];
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) acc[i] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
    for (int w0 = 0; w0 < NW; w0 += 4) {
        if (wave >= w0 && wave < w0 + 4) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                f4 v = o[dt];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (WIDE) v[i] = fmaf(o2[dt][i], 1.0f / A4_LO, v[i]);
                    else v[i] = ror8_add(v[i] * lo_unit);
                }
                if (col < rows) *(f4 *)&mo[wave - w0][col][16 * dt + 4 * g] = v * 16.0f;
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < SLOTS; ++i) {
            const int e4 = i * 64 * NW + tid, h = e4 / (D / 4), dd = e4 % (D / 4) * 4;
            if (h >= rows) break;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const f4 v = *(const f4 *)&mo[w][h][dd];
                const float f = sc[h][w0 + w];
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(v[j], f, acc[i][j]);
            }
        }
        if (w0 + 4 < NW) __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {  // 8 lanes hold a Q8_0 block
        const int e4 = i * 64 * NW + tid, h = e4 / (D / 4), dd = e4 % (D / 4) * 4;
        if (h >= rows) break;
        const size_t row = head_of(h);
        if (whole) {
            const float r = linv[h];
            const float y[4] = {acc[i][0] * r, acc[i][1] * r, acc[i][2] * r, acc[i][3] * r};
            kv4_store(y, row * D + dd, e4 & 7, attn, qs, qd8, bsum, ROWS ? nullptr : tq, td,
                      qheads * D, qi);
        } else {
            *(f4 *)(ws_o + (row * ns + sp) * D + dd) = acc[i];
        }
    }
}

// ---------------------------------------------------------------------------
// The chunks' states of a (query, head) to its output: a workgroup per 32 dims
// (one Q8_0 block), 8 lanes a state, G states at once, at most 8 G in all, so
// that every load is in flight at once: 3.9-4.0 us, a launch, one round trip and the
// stores.  tq/td (optional): the Q8_0 also
// operand-tiled (q8_tiled_byte).
// ---------------------------------------------------------------------------
template <int G>
__global__ void __launch_bounds__(8 * G) k_kv4_merge(
    int qheads, int hdim, int ns, const int *__restrict__ ctx_dev, const int *__restrict__ parts,
    const float *__restrict__ ws_u, const float *__restrict__ ws_m,
    const float *__restrict__ ws_l, const float *__restrict__ ws_o, float *__restrict__ attn,
    int8_t *__restrict__ qs, uint16_t *__restrict__ d, int16_t *__restrict__ bsum,
    int8_t *__restrict__ tq, uint16_t *__restrict__ td) {
    constexpr int W = G / 8;  // wavefronts
    __shared__ float red_m[W], red_l[W];
    __shared__ f4 red_o[W][8];
    const int nb = hdim / 32, h = blockIdx.x / nb, blk = blockIdx.x % nb, qi = blockIdx.y;
    const int tid = threadIdx.x, l8 = tid & 7, grp = tid >> 3, wave = tid >> 6;
    const size_t base = ((size_t)qi * qheads + h) * ns;
    const int each = (ns + G - 1) / G;
    const int have = !parts ? ns : ctx_dev[qi] > 0 ? parts[qi] : 0;  // states that were written
    if (parts && have == 1) return;  // its workgroup wrote the output
    const float unit = ws_u[(size_t)qi * qheads + h];
    f4 o[8];
    float m[8], l[8], mx = -INFINITY;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        m[k] = -INFINITY;
        if (k < each && grp + k * G < ns) {
            const size_t i = base + grp + k * G;
            m[k] = ws_m[i];
            l[k] = ws_l[i];
            o[k] = *(const f4 *)(ws_o + i * hdim + 32 * blk + 4 * l8);
        }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        m[k] = grp + k * G < have ? m[k] : -INFINITY;
        mx = fmaxf(mx, m[k]);
    }
    mx = fmaxf(mx, dpp_f<DPP_ROR8>(mx));
    mx = fmaxf(mx, swap16_f(mx));
    mx = fmaxf(mx, swap32_f(mx));
    if constexpr (W > 1) {
        if ((tid & 63) == 0) red_m[wave] = mx;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) mx = fmaxf(mx, red_m[w]);
    }
    f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        if (m[k] == -INFINITY) continue;  // none, or an empty chunk (its output unwritten)
        const float w = __builtin_amdgcn_exp2f((m[k] - mx) * unit);
        sum = fmaf(l[k], w, sum);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = fmaf(o[k][i], w, acc[i]);
    }
    auto across = [](float v) {
        v = ror8_add(v);
        v += swap16_f(v);
        return v + swap32_f(v);
    };
    sum = across(sum);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = across(acc[i]);
    if constexpr (W > 1) {
        if ((tid & 63) < 8) red_o[wave][l8] = acc;
        if ((tid & 63) == 0) red_l[wave] = sum;
        __syncthreads();
        acc = red_o[0][l8];
        sum = red_l[0];
#pragma unroll
        for (int w = 1; w < W; ++w) {
            acc += red_o[w][l8];
            sum += red_l[w];
        }
    }
    if (tid >= 8) return;
    const float r = mx == -INFINITY ? 0.0f : 1.0f / sum;  // no context: zeros
    const float y[4] = {acc[0] * r, acc[1] * r, acc[2] * r, acc[3] * r};
    const size_t off = ((size_t)qi * qheads + h) * hdim + 32 * blk + 4 * l8;
    kv4_store(y, off, l8, attn, qs, d, bsum, tq, td, qheads * hdim, qi);
}

// ---------------------------------------------------------------------------
// page copies: grid (pieces of a page, moves, pools); the pools' addresses and
// the moves travel in the kernel's arguments, so the call needs no upload.  Four
// loads of a thread are in flight.  ONCE: a call past the 256 MB cache goes past it
// both ways (500 pages of 64 KB in 16 pools, 1.05 GB read and written: 178 us, 5.9
// TB/s, else 190, and 209 with a load at a time; 700 of 36 KB 156, else 167), a
// smaller one may find its pages there (100 of 18 KB in 16 pools 12.2, else 10.9).
// 3 pages of 18 KB in 56 pools 3.1 us.
// ---------------------------------------------------------------------------
template <class T, bool ONCE>
__global__ void __launch_bounds__(256) k_kv_copy(KvMoves mv, size_t page_bytes) {
    uint8_t *pool = mv.pool[blockIdx.z];
    const T *src = (const T *)(pool + (size_t)mv.src[blockIdx.y] * page_bytes);
    T *dst = (T *)(pool + (size_t)mv.dst[blockIdx.y] * page_bytes);
    const size_t n = page_bytes / sizeof(T), step = (size_t)gridDim.x * 256;
    auto get = [&](size_t i) { return ONCE ? __builtin_nontemporal_load(src + i) : src[i]; };
    auto put = [&](T v, size_t i) {
        if constexpr (ONCE) __builtin_nontemporal_store(v, dst + i);
        else dst[i] = v;
    };
    size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    for (; i + 3 * step < n; i += 4 * step) {
        T t[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) t[k] = get(i + k * step);
#pragma unroll
        for (int k = 0; k < 4; ++k) put(t[k], i + k * step);
    }
    for (; i < n; i += step) put(get(i), i);
}

// ---------------------------------------------------------------------------
// launchers
// ---------------------------------------------------------------------------
#define KV4_DIM(hdim, CALL)       \
    switch (hdim) {               \
        case 32: CALL(32); break; \
        case 64: CALL(64); break; \
        case 96: CALL(96); break; \
        default: CALL(128); break; \
    }

void launch_rope_kv4(const float *qkv, int ldqkv, int ntok, int qheads, int hdim, int pos0,
                     int pos_step, int max_pos, const int *ctx_dev, const float *rc,
                     const float *rs, float *q_out, const Kv4Cache &c, hipStream_t st,
                     bool clamp) {
    if (ntok <= 0) return;
    const int limit = (int)min((long long)max_pos, (long long)c.max_pages << c.shift);
    const int qy = (qheads * hdim / 2 + 2 * hdim - 1) / (2 * hdim);
    const bool wide =
        ldqkv % 4 == 0 && (((uintptr_t)qkv | (uintptr_t)rc | (uintptr_t)rs) & 15) == 0;
    const dim3 grid(kv4_units(ntok, pos0, pos_step), c.kvheads + qy);
#define CALL(DIM)                                                                               \
    SI_LAUNCH((k_kv4_append<DIM, false>), grid, dim3(2 * DIM), 0, st, qkv, ldqkv, nullptr,      \
              nullptr, qheads, ntok, pos0, pos_step, limit, ctx_dev, rc, rs, q_out, wide, clamp, c)
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
              pos0, pos_step, limit, ctx_dev, nullptr, nullptr, nullptr, false, false, c)
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

// How a call runs: wavefronts a workgroup, the most chunks of a context, and the
// workgroups that the GPU holds at once.  By base, the (query, KV head) pairs or
// blocks of 16 rows, and the steps of 128 positions of the longest context (device
// contexts: of max_ctx);
// us a call in a graph, split | whole in four | in eight, contexts equal (1/16 to all of
// the longest):
//   - whole in four wavefronts up to 4 steps: the merge and its launch cost about 4 us.
//     28/4 heads of 128, 1 query of 512 8.7 | 7.7 | 8.0, 48 of 384 13.0 | 7.4 | 7.7.
//   - with at most one workgroup a CU, whole in eight up to the steps below: they share
//     a context's steps, and step faster than three wavefronts a SIMD.  28/4 heads of
//     128: 16 of 1536 13.1 | 16.6 | 14.2; 48 of 2048 21.8 | 22.1 | 18.4; 64 of 4096 36.0 | 39.0 |
//     31.1 (25.5 | 37.2 | 28.3), of 8192 64.1 | 72.7 | 57.9 (39.5 | 69.7 | 50.2).  14/2 of 64: 64 of
//     3000 15.7 | 22.5 | 16.9 (13.7 | 21.4 | 16.2); 128 of 4096 26.3 | 29.5 | 21.5 (19.4 | 28.4 |
//     20.7).  8/8 of 32: 6 of 1536 8.9 | 10.1 | 8.5; 32 of 4096 19.5 | 24.4 | 17.0 (16.2 | 23.5 |
//     16.4).  One query's border is set by calls one by one, whose second launch the host
//     is late with: 14/2 of 64, 1 of 1024 9.6 | 8.9 | 8.3 from Python, 7.9 | 8.9 | 8.3 in a graph;
//     28/4 of 128, 1 of 768 8.5 | 9.6 | 9.2 there, of 1024 8.8 | 10.9 | 10.4.
//   - with more, whole in four up to 5 + base / 32 steps: 28/4 heads of 128, 80 queries of 1024
//     26.3 | 17.0 | 21.3, of 2048 34.0 | 28.0 | 33.0 (28.3 | 25.2 | 22.8), of 3000 41.6 | 38.7 |
//     43.8 (32.0 | 35.0 | 29.7); 128 of 2048 46.2 | 30.5 | 36.0, of 4096 68.9 | 58.6 | 63.5.
//   - from `slots` pairs on (and not by their lengths) whole in four: contexts of about one
//     length; one far longer than the others is walked by its one workgroup.
//   - else split into chunks: as many as fill the GPU (three, four or five workgroups a
//     CU by their registers), or fill it twice where they would be two or fewer a pair,
//     too coarse to end together: once | twice, 93 to 6000 positions (6000), 24/8 heads
//     of 96: 40 queries 34.9 | 34.2 (49.1 | 46.5), 48 36.6 | 34.7 (51.5 | 52.0), 75 63.2 |
//     50.2 (84.7 | 81.5); 26 26.9 | 26.0 (35.3 | 34.1).  A context on the device may get
//     twice its share, which the kernel uses as they are ragged.
struct A4Plan {
    int nw, ns, slots;
};
static A4Plan a4_plan(int hdim, long long base, int max_ctx, bool ragged) {
    const long long steps = ((long long)max_ctx + 4 * A4_GROUP - 1) / (4 * A4_GROUP);
    int slots = hdim > 64 ? 768 : hdim > 32 ? 1024 : 1280;
    if (base >= slots || steps <= 4) return {4, 1, slots};
    if (base <= 256 ? steps <= 4 + 256 / hdim + base / 8 : steps <= 5 + base / 32)
        return {base <= 256 ? 8 : 4, 1, slots};
    if (base > slots * 2 / 5) slots *= 2;
    const long long want = (slots + base - 1) / base * (ragged ? 2 : 1);
    return {4, (int)min(min(steps, want), 256ll), slots};
}

// Whether a prompt's pages are read into fp16 rows for the prefill kernel, which
// unpacks nothing and takes 32 rows a tile, but walks a tile's context in one
// workgroup: it pays once its tiles fill the GPU, whatever the context.  Both ways (us a
// call in a graph, over the pages | by rows, after 300, 1500 and 6000 positions): 28/4
// heads of 128, 16 queries 9 | 15, 12 | 31, 19 | 91; 256 15 | 19, 29 | 34, 86 | 93; 333 17 |
// 21, 37 | 41, 108 | 107; 512 26 | 25, 53 | 46, 156 | 130; 2048 130 | 101, 220 | 171, 559 | 428.
// 14/2 of 64, 512 11 | 14, 21 | 22, 54 | 52; 768 16 | 16, 28 | 26, 77 | 68.  16/1 of 128, 600 21 |
// 23, 40 | 38, 117 | 100.  24/8 of 96, 512 18 | 21, 34 | 37, 95 | 101; 1000 37 | 36, 67 | 62, 184
// | 167.  8/8 of 32, 1024 12 | 14, 19 | 21, 42 | 46; 2000 22 | 20, 32 | 29, 81 | 65.
// (Past 2^26 positions the rows would be a launch of 2^31 threads and more.)
static bool kv4_by_rows(int qheads, int nq, int ctx_step, int max_ctx) {
    return ctx_step == 1 && (long long)nq * qheads > 9000 && max_ctx <= 1 << 26;
}

// Workgroups of a call that splits no context
static long long a4_base(int qheads, int kvheads, int nq, int ctx_step) {
    const long long rows = (long long)nq * (qheads / kvheads);
    return kvheads * (ctx_step && nq > 1 ? (rows + 15) / 16 : (long long)nq);
}

size_t attn_kv4_workspace(int qheads, int kvheads, int hdim, int nq, int ctx_step, int max_ctx) {
    if (kv4_by_rows(qheads, nq, ctx_step, max_ctx))
        return (size_t)max_ctx * kvheads * hdim * 2 * sizeof(uint16_t);
    const long long base = a4_base(qheads, kvheads, nq, ctx_step);
    const int ns = max(a4_plan(hdim, base, max_ctx, false).ns,
                       ctx_step ? 1 : a4_plan(hdim, base, max_ctx, true).ns);
    if (ns == 1) return 0;
    return (size_t)nq * qheads * (ns * (size_t)(hdim + 2) + 1) * sizeof(float) +
           (size_t)nq * sizeof(int);
}

void launch_attention_kv4(const float *q, int nq, int qheads, int hdim, const Kv4Cache &c,
                          const int *ctx_dev, int ctx0, int ctx_step, int max_ctx, float *attn,
                          int8_t *qs, uint16_t *d, int16_t *bsum, void *ws, hipStream_t st,
                          int8_t *tq, uint16_t *td) {
    if (nq <= 0) return;
    if (kv4_by_rows(qheads, nq, ctx_step, max_ctx)) {
        uint16_t *k = (uint16_t *)ws, *v = k + (size_t)max_ctx * c.kvheads * hdim;
        launch_kv4_read(c, ctx0 - 1 + nq, hdim, 0, 1, nullptr, k, v, st);
        launch_attn_prefill(q, nq, qheads, c.kvheads, hdim, ctx0 - 1, k, v, attn, qs, d, bsum, st,
                            true);
        return;
    }
    const long long base = a4_base(qheads, c.kvheads, nq, ctx_step);
    const A4Plan plan = a4_plan(hdim, base, max_ctx, ctx_dev != nullptr);
    const int ns = plan.ns, slots = plan.slots, step = plan.nw * A4_GROUP;
    const int chunk = ((max_ctx + ns - 1) / ns + step - 1) / step * step;
    const AttnParts pt(ws, (size_t)nq * qheads * ns, hdim);
    // contexts on the device: a list of chunks, its length made on the GPU
    float *unit = pt.l + (size_t)nq * qheads * ns;
    int *parts = ns > 1 && ctx_dev ? (int *)(unit + (size_t)nq * qheads) : nullptr;
    const long long items =
        parts ? min((long long)slots / c.kvheads + nq, (long long)nq * ns) : base / c.kvheads;
    const dim3 grid(c.kvheads, (unsigned)items, parts ? 1 : ns);
    const bool rows = ctx_step && nq > 1, wide = qheads / c.kvheads > 8, page16 = c.shift == 4;
#define CALL3(DIM, M, P, NW)                                                                    \
    SI_LAUNCH((k_attn_kv4<DIM, M, P, NW>), grid, dim3(64 * NW), 0, st, q, qheads, c, ctx_dev,    \
              ctx0, ctx_step, nq, max_ctx, ns, chunk, slots, softmax_scale2(hdim), parts, unit, \
              pt.m, pt.l, pt.o, attn, qs, d, bsum, tq, td)
#define CALL2(DIM, M)                                                  \
    if (plan.nw == 4 && page16) CALL3(DIM, M, true, 4);                \
    else if (plan.nw == 4) CALL3(DIM, M, false, 4);                    \
    else if (page16) CALL3(DIM, M, true, 8);                           \
    else CALL3(DIM, M, false, 8)
#define CALL(DIM)                           \
    if (rows) { CALL2(DIM, A4_ROWS); }      \
    else if (wide) { CALL2(DIM, A4_WIDE); } \
    else { CALL2(DIM, A4_NARROW); }
    KV4_DIM(hdim, CALL)
#undef CALL
#undef CALL2
#undef CALL3
    if (ns == 1) return;
    const dim3 blocks(qheads * (hdim / 32), nq);
#define CALL(G)                                                                                  \
    SI_LAUNCH(k_kv4_merge<G>, blocks, dim3(8 * G), 0, st, qheads, hdim, ns, ctx_dev, parts, unit, \
              pt.m, pt.l, pt.o, attn, qs, d, bsum, tq, td)
    if (ns <= 64) CALL(8);
    else CALL(32);
#undef CALL
}

void launch_kv_copy(const KvMoves &mv, int npools, int nmoves, size_t page_bytes, bool wide,
                    bool once, hipStream_t st) {
    const size_t unit = wide ? 16 : 1;
    const size_t want = (page_bytes / unit + 256 * 4 - 1) / (256 * 4);
    const dim3 grid((unsigned)min(want, (size_t)64), nmoves, npools);
    if (wide && once) SI_LAUNCH((k_kv_copy<u4, true>), grid, dim3(256), 0, st, mv, page_bytes);
    else if (wide) SI_LAUNCH((k_kv_copy<u4, false>), grid, dim3(256), 0, st, mv, page_bytes);
    else SI_LAUNCH((k_kv_copy<uint8_t, false>), grid, dim3(256), 0, st, mv, page_bytes);
}
}  // namespace si
