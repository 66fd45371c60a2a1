// si_step.hip -- the bookkeeping of a ragged step over a paged cache, on the GPU: page
// lists and slot maps from the sequences' lengths, and the RoPE + K/V append by slot.
// No counterpart in the reference (one sequence, one contiguous cache,
// qwen_one_layer.c:262-266).
#include "si_device.hpp"
#include "si_kernels.hpp"

namespace si {

// ---------------------------------------------------------------------------
// Page lists and slot maps (si_kv_step)
//
// A sequence's step is known from its own numbers: positions have + add, pages
// ceil((have + add) / page) - taken more, pages that lie behind the window of position
// have given back.  Three prefix sums over the sequences (rows, pages taken, pages given
// back) then say where each writes.
// ---------------------------------------------------------------------------
struct StepSeq {
    int have, add, taken, gone;  // as given, within their ranges
    int more, now;               // pages taken in this step; pages given back after it
    bool ended, bad;
};

__device__ __forceinline__ StepSeq step_seq(const KvStep &a, int i) {
    StepSeq s;
    const long long ps = 1ll << a.shift;
    const int have = a.have[i], add = max(a.add[i], 0);
    s.ended = have < 0;
    s.have = max(have, 0);
    s.taken = min(max(a.held_in[2 * i], 0), a.max_pages);
    s.gone = min(max(a.held_in[2 * i + 1], 0), max(s.taken - a.kept, 0));
    s.bad = !s.ended && ((long long)s.have + add > a.max_pages * ps || s.have > s.taken * ps);
    s.add = s.ended || s.bad ? 0 : add;
    const int need = (int)(((long long)s.have + s.add + ps - 1) >> a.shift);
    s.more = s.ended || s.bad ? 0 : max(need - s.taken, 0);
    // (have - window + 1 positions lie behind every window from here on)
    const int behind = (int)((max((long long)s.have - a.window + 1, 0ll)) >> a.shift);
    s.now = s.ended || s.bad ? s.gone : max(s.gone, min(behind, s.taken) - a.kept);
    return s;
}
// ids that the sequence puts back into the ring, in the order of its list
__device__ __forceinline__ int step_back(const KvStep &a, const StepSeq &s) {
    return s.ended ? min(a.kept, s.taken) + max(s.taken - a.kept - s.gone, 0) : s.now - s.gone;
}
__device__ __forceinline__ int step_back_page(const KvStep &a, const StepSeq &s, int k) {
    if (!s.ended) return a.kept + s.gone + k;
    const int first = min(a.kept, s.taken);
    return k < first ? k : a.kept + s.gone + k - first;
}

// exclusive prefix sum over the workgroup of one value a thread; total: its sum
__device__ __forceinline__ long long block_scan(long long v, long long *red, long long &total) {
    long long x = v;
    for (int d = 1; d < 64; d <<= 1) {
        const long long y = __shfl_up(x, d, 64);
        if ((int)(threadIdx.x & 63) >= d) x += y;
    }
    __syncthreads();  // red may still be read from the scan before
    if ((threadIdx.x & 63) == 63) red[threadIdx.x >> 6] = x;
    __syncthreads();
    long long base = 0;
    total = 0;
    for (int w = 0; w < (int)(blockDim.x >> 6); ++w) {
        if (w < (int)(threadIdx.x >> 6)) base += red[w];
        total += red[w];
    }
    return base + x - v;
}

constexpr int STEP_T = 1024;
__global__ void __launch_bounds__(STEP_T) k_kv_step(KvStep a) {
    __shared__ long long red[STEP_T / 64];
    const int tid = threadIdx.x;
    const int per = (a.nseq + STEP_T - 1) / STEP_T;
    const int i0 = min(tid * per, a.nseq), i1 = min(i0 + per, a.nseq);
    const int begin = min(max(a.free_in[0], 0), a.npages - 1);
    const int count = min(max(a.free_in[1], 0), a.npages);
    long long rows = 0, more = 0, back = 0, bad = 0;
    for (int i = i0; i < i1; ++i) {
        const StepSeq s = step_seq(a, i);
        rows += s.add;
        more += s.more;
        back += step_back(a, s);
        bad += s.bad;
    }
    long long nrows, nmore, nback, nbad;
    rows = block_scan(rows, red, nrows);
    more = block_scan(more, red, nmore);
    back = block_scan(back, red, nback);
    block_scan(bad, red, nbad);
    const int code = (nrows > a.max_rows ? 1 : 0) | (nmore > count ? 2 : 0) | (nbad ? 4 : 0);
    const auto wrap = [&](long long k) { return (int)((begin + k) % a.npages); };
    for (int i = i0; i < i1; ++i) {
        const StepSeq s = step_seq(a, i);
        int *list = a.pages + (size_t)i * a.max_pages;
        if (code) {
            a.start[i] = a.taken[i] = 0;
            a.ctx[i] = s.have;
            a.held_out[2 * i] = s.taken;
            a.held_out[2 * i + 1] = s.gone;
            continue;
        }
        a.start[i] = (int)rows;
        a.taken[i] = (int)more;
        a.ctx[i] = s.ended ? 0 : s.have + s.add;
        for (int k = 0; k < s.more; ++k) list[s.taken + k] = a.ring[wrap(more + k)];
        const int nb = step_back(a, s);
        for (int k = 0; k < nb; ++k)
            a.ring[wrap(count + back + k)] = list[step_back_page(a, s, k)];
        a.held_out[2 * i] = s.ended ? 0 : s.taken + s.more;
        a.held_out[2 * i + 1] = s.ended ? 0 : s.now;
        rows += s.add;
        more += s.more;
        back += nb;
    }
    if (tid == 0) {
        a.start[a.nseq] = code ? 0 : (int)nrows;
        a.taken[a.nseq] = code ? 0 : (int)nmore;
        a.free_out[0] = code ? begin : wrap(nmore);
        a.free_out[1] = code ? count : (int)min(count - nmore + nback, (long long)a.npages);
        a.status[0] = code;
        a.status[1] = (int)min(nrows, (long long)INT_MAX);
        a.status[2] = (int)min(nmore, (long long)INT_MAX);
        a.status[3] = code ? 0 : (int)nback;
    }
    __syncthreads();
    const int n = code ? 0 : (int)nrows;
    for (int r = tid; r < a.max_rows; r += STEP_T) {
        int seq = -1, pos = -1;
        long long slot = -1;
        if (r < n) {
            int lo = 0, hi = a.nseq;  // start[lo] <= r < start[hi]
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (a.start[mid] <= r) lo = mid;
                else hi = mid;
            }
            seq = lo;
            pos = a.ctx[lo] - a.start[lo + 1] + r;
            const int id = a.pages[(size_t)lo * a.max_pages + (pos >> a.shift)];
            slot = ((long long)min(max(id, 0), a.npages - 1) << a.shift) |
                   (pos & ((1 << a.shift) - 1));
        }
        a.seq[r] = seq;
        a.pos[r] = pos;
        a.slot[r] = slot;
    }
}

void launch_kv_step(const KvStep &a, hipStream_t st) {
    SI_LAUNCH(k_kv_step, dim3(1), dim3(STEP_T), 0, st, a);
}

// ---------------------------------------------------------------------------
// RoPE and the K/V append by slot (si_rope_kv_append_rows)
//
// The arithmetic and the bits of k_rope_kv: a' = a c - b s, b' = b c + a s, and the fp16
// narrowing.  Memory bounds it; a thread takes four neighbouring pairs of a head (16-byte
// loads and stores of q|k|v and q, 8-byte stores of the cache), or four values of V's two
// halves.
// ---------------------------------------------------------------------------
constexpr int ROWS_T = 256;
__global__ void __launch_bounds__(ROWS_T) k_rope_kv_rows(
    const float *__restrict__ qkv, int ldqkv, int qheads, int kvheads, int hdim, int max_pos,
    const int *__restrict__ row_pos, const long long *__restrict__ slot,
    const float *__restrict__ rc, const float *__restrict__ rs, float *__restrict__ q_out,
    uint16_t *__restrict__ kc, uint16_t *__restrict__ vc, long long pool_rows) {
    const int t = blockIdx.x, half = hdim >> 1, quads = half / 4;
    const int j = blockIdx.y * ROWS_T + threadIdx.x;
    if (j >= (qheads + 2 * kvheads) * quads) return;
    const int pos = row_pos[t];
    const long long at = slot[t];
    // (device data: a row without a position or a place is left as it is)
    if (pos < 0 || pos >= max_pos || at < 0 || at >= pool_rows) return;
    const int h = j / quads, i = 4 * (j - h * quads);
    const float *src = qkv + (size_t)t * ldqkv + h * hdim + i;
    float a[4], b[4], x[4], y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] = src[e], b[e] = src[half + e];
    if (h < qheads + kvheads) {
        const float4 c4 = *(const float4 *)(rc + (size_t)pos * half + i);
        const float4 s4 = *(const float4 *)(rs + (size_t)pos * half + i);
        const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[e] = __fsub_rn(__fmul_rn(a[e], c[e]), __fmul_rn(b[e], s[e]));
            y[e] = __fadd_rn(__fmul_rn(b[e], c[e]), __fmul_rn(a[e], s[e]));
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = a[e], y[e] = b[e];
    }
    if (h < qheads) {
        float *q = q_out + ((size_t)t * qheads + h) * hdim + i;
        *(float4 *)q = make_float4(x[0], x[1], x[2], x[3]);
        *(float4 *)(q + half) = make_float4(y[0], y[1], y[2], y[3]);
        return;
    }
    const bool k = h < qheads + kvheads;
    const int g = h - qheads - (k ? 0 : kvheads);
    uint16_t *to = (k ? kc : vc) + ((size_t)at * kvheads + g) * hdim + i;
    ushort4 lo, hi;
    lo.x = f2h(x[0]), lo.y = f2h(x[1]), lo.z = f2h(x[2]), lo.w = f2h(x[3]);
    hi.x = f2h(y[0]), hi.y = f2h(y[1]), hi.z = f2h(y[2]), hi.w = f2h(y[3]);
    *(ushort4 *)to = lo;
    *(ushort4 *)(to + half) = hi;
}

void launch_rope_kv_rows(const float *qkv, int ldqkv, int rows, int qheads, int kvheads, int hdim,
                         int max_pos, const int *pos, const long long *slot, const float *rc,
                         const float *rs, float *q_out, uint16_t *kc, uint16_t *vc,
                         long long pool_rows, hipStream_t st) {
    const int quads = (qheads + 2 * kvheads) * (hdim / 8);
    SI_LAUNCH(k_rope_kv_rows, dim3(rows, (quads + ROWS_T - 1) / ROWS_T), dim3(ROWS_T), 0, st, qkv,
              ldqkv, qheads, kvheads, hdim, max_pos, pos, slot, rc, rs, q_out, kc, vc, pool_rows);
}

}  // namespace si
