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
            const int pos = ctx_dev ? ctx_dev[x] - 1 : pos0;
            seq = x;
            base = pos & ~7;
            lo = pos & 7;
            t0 = x - lo;
            hi = pos >= 0 && pos < limit ? lo + 1 : lo;  // device contexts: not host-checked
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
// attention: a workgroup per (query, KV head), 256 positions at a time with the
// running maximum and sum of the softmax
// ---------------------------------------------------------------------------
template <int D>
__global__ void __launch_bounds__(256) k_attn_kv4(const float *__restrict__ q, int qheads,
                                                  Kv4Cache c, const int *__restrict__ ctx_dev,
                                                  int ctx0, int ctx_step, int max_ctx,
                                                  float scale2, float *__restrict__ attn) {
    constexpr int NB = D / 32;
    __shared__ float ql[16 * D], p[16][256], red[4];
    const int g = blockIdx.x, qi = blockIdx.y, tid = threadIdx.x, per = qheads / c.kvheads;
    const int seq = ctx_step ? 0 : qi, page_size = 1 << c.shift;
    const int ctx = min(ctx_dev ? ctx_dev[qi] : ctx0 + qi * ctx_step, max_ctx);
    const size_t hb = (size_t)kv4_head_bytes(D, page_size);
    const float *qrow = q + ((size_t)qi * qheads + g * per) * D;
    for (int i = tid; i < per * D; i += 256) ql[i] = qrow[i];
    __syncthreads();
    float m[16], l[16], o[16];  // o: dim tid of each head (tid < D)
    for (int h = 0; h < 16; ++h) m[h] = -INFINITY, l[h] = o[h] = 0.0f;
    for (int s0 = 0; s0 < ctx; s0 += 256) {
        const int pos = s0 + tid;
        float s[16];
        for (int h = 0; h < 16; ++h) s[h] = 0.0f;
        if (pos < ctx) {
            const int i = pos & (page_size - 1);
            const uint8_t *kp = c.k + ((size_t)c.page_of(seq, pos) * c.kvheads + g) * hb;
            for (int b = 0; b < NB; ++b) {
                const float d = h2f_fast(*(const uint16_t *)(kp + kv4_scale(D, page_size, i, b))) * 16.0f;
                for (int gg = 0; gg < 4; ++gg) {
                    const uint32_t w = *(const uint32_t *)(kp + kv4_k_dword(D, i, 4 * b + gg));
                    for (int e = 0; e < 8; ++e) {
                        const float x = (float)((int)(w >> (4 * e) & 15) - 8) * d;
                        for (int h = 0; h < 16; ++h)
                            if (h < per) s[h] = fmaf(x, ql[h * D + 32 * b + 8 * gg + e], s[h]);
                    }
                }
            }
        }
        for (int h = 0; h < 16; ++h) {
            if (h >= per) break;
            const float t = pos < ctx ? s[h] * scale2 : -INFINITY;
            float mx = wave_max(t);
            __syncthreads();
            if ((tid & 63) == 0) red[tid >> 6] = mx;
            __syncthreads();
            mx = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), m[h]);
            const float ref = mx == -INFINITY ? 0.0f : mx;
            const float al = __builtin_amdgcn_exp2f(m[h] - ref), pp = __builtin_amdgcn_exp2f(t - ref);
            p[h][tid] = pp;
            const float sum = wave_sum(pp);
            __syncthreads();
            if ((tid & 63) == 0) red[tid >> 6] = sum;
            __syncthreads();
            l[h] = l[h] * al + (red[0] + red[1] + red[2] + red[3]);
            o[h] *= al;
            m[h] = mx;
        }
        __syncthreads();
        if (tid < D) {
            const int n = min(ctx - s0, 256);
            for (int j = 0; j < n; ++j) {
                const int ps = s0 + j, i = ps & (page_size - 1);
                const uint8_t *vp = c.v + ((size_t)c.page_of(seq, ps) * c.kvheads + g) * hb;
                const uint32_t w = *(const uint32_t *)(vp + kv4_v_dword(D, i >> 3, tid));
                const float d = h2f_fast(*(const uint16_t *)(vp + kv4_scale(D, page_size, i, tid >> 5))) * 16.0f;
                const float x = (float)((int)(w >> (4 * (i & 7)) & 15) - 8) * d;
                for (int h = 0; h < 16; ++h)
                    if (h < per) o[h] = fmaf(p[h][j], x, o[h]);
            }
        }
        __syncthreads();
    }
    if (tid < D)
        for (int h = 0; h < 16; ++h)
            if (h < per)
                attn[((size_t)qi * qheads + g * per + h) * D + tid] = ctx > 0 ? o[h] / l[h] : 0.0f;
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

size_t attn_kv4_workspace(int, int, int, int, int, int) { return 0; }

void launch_attention_kv4(const float *q, int nq, int qheads, int hdim, const Kv4Cache &c,
                          const int *ctx_dev, int ctx0, int ctx_step, int max_ctx, float *attn,
                          int8_t *qs, uint16_t *d, int16_t *bsum, void *, size_t,
                          hipStream_t st) {
    if (nq <= 0) return;
#define CALL(DIM)                                                                              \
    SI_LAUNCH((k_attn_kv4<DIM>), dim3(c.kvheads, nq), dim3(256), 0, st, q, qheads, c, ctx_dev, \
              ctx0, ctx_step, max_ctx, softmax_scale2(hdim), attn)
    KV4_DIM(hdim, CALL)
#undef CALL
    if (qs) launch_quantize_q8_rows(attn, nq, qheads * hdim, qs, d, bsum, st);
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
