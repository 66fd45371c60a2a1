// si_step.hip -- the bookkeeping of a ragged step over a paged cache, on the GPU: page
// lists and slot maps from the sequences' lengths, and the RoPE + K/V append by slot.
// No counterpart in the reference (one sequence, one contiguous cache,
// qwen_one_layer.c:262-266).
#include <algorithm>

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
//
// Latency bounds it: a step's numbers are 16 bytes a sequence and 16 a row (4000 sequences and as
// many rows 1.7 MB, 0.3 us at a copy's rate), but a chain of dependent steps lies between them:
// lengths, the sums over a wavefront and the workgroup, a row's search for its sequence, its
// page's id, the stores.  One small workgroup takes 3.2 us, 4000 sequences of up to 5 rows and 40
// pieces of 2000 10 us over many (12 where a row had up to four sequences to walk).  (Each
// sequence's rows written by its own thread took 22 us for 200 sequences and 333 for the 4000.)
// ---------------------------------------------------------------------------
struct StepSeq {
    int have, add, taken, gone;  // as given (add: 0 of a sequence without rows)
    int more, now;               // pages taken in this step; pages given back after it
    bool ended, bad;             // (bad: the step is refused, only what was given is of use)
};

__device__ __forceinline__ StepSeq step_seq(const KvStep &a, int i) {
    StepSeq s;
    const long long ps = 1ll << a.shift;
    const int add = max(a.add[i], 0);
    s.have = a.have[i];
    s.taken = a.held_in[2 * i];
    s.gone = a.held_in[2 * i + 1];
    s.ended = s.have < 0;
    const int taken = min(max(s.taken, 0), a.max_pages);
    // (have - window + 1 positions lie behind every window from here on; an ended sequence may
    // have given back any of its pages)
    const int behind = (int)((max((long long)s.have - a.window + 1, 0ll)) >> a.shift);
    s.now = max((s.ended ? taken : min(behind, taken)) - a.kept, 0);
    // (counts that no step left; rows from a have whose window reaches pages that were given back
    // would see others' pages, or be written to them)
    s.bad = taken != s.taken || (unsigned)s.gone > (unsigned)s.now ||
            (!s.ended && ((long long)s.have + add > a.max_pages * ps || s.have > taken * ps));
    s.add = s.ended || s.bad ? 0 : add;
    const int need = (int)(((long long)s.have + s.add + ps - 1) >> a.shift);
    s.more = s.ended || s.bad ? 0 : max(need - taken, 0);
    return s;
}
// The ring's state.  One outside its ranges is no step's: what its ids are is not known, so that
// the step is refused and the ring empty from then on.
struct StepRing {
    int begin, count;
    bool bad;
};
__device__ __forceinline__ StepRing step_ring(const KvStep &a) {
    const int begin = a.free_in[0], count = a.free_in[1];
    const bool bad = begin < 0 || begin >= a.npages || count < 0 || count > a.npages;
    return {bad ? 0 : begin, bad ? 0 : count, bad};
}
// a sequence's state after the step (of a refused one as given, whatever it is), and the ring's
__device__ __forceinline__ void step_state(const KvStep &a, int i, const StepSeq &s, int code) {
    a.held_out[2 * i] = code ? s.taken : s.ended ? 0 : s.taken + s.more;
    a.held_out[2 * i + 1] = code ? s.gone : s.ended ? 0 : s.now;
}
__device__ __forceinline__ void ring_state(const KvStep &a, const StepRing &ring, int code,
                                           long long more, long long back) {
    const long long to = ring.begin + more;  // (of a step that succeeds at most npages more)
    a.free_out[0] = code ? ring.begin : (int)(to >= a.npages ? to - a.npages : to);
    a.free_out[1] = code ? ring.count : (int)(ring.count - more + back);
}
// whether that is written beside the state that this step starts from, not over it
__host__ __device__ __forceinline__ bool apart(const KvStep &a) {
    return a.held_out != a.held_in && a.free_out != a.free_in;
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

// what the sequences of a thread add up to, before (of) and in (the sums) the workgroup
struct StepSums {
    // (held: pages in the lists before the step; a sequence that is refused counts as one of
    // more pages than there can be)
    long long rows = 0, more = 0, back = 0, held = 0;
    __device__ __forceinline__ void add(const KvStep &a, const StepSeq &s) {
        rows += s.add;
        more += s.more;
        back += s.bad ? 0 : step_back(a, s);
        held += s.bad ? 1ll << 40 : s.taken - s.gone;
    }
    __device__ __forceinline__ void add(const StepSums &x) {
        rows += x.rows;
        more += x.more;
        back += x.back;
        held += x.held;
    }
};

constexpr int STEP_T = 1024, STEP_FEW = 256;  // threads of a workgroup; of one for few rows

// exclusive prefix sums over the workgroup's threads (of rows, more and back); the totals
template <int T>
__device__ __forceinline__ void step_scan(StepSums &v, StepSums &total) {
    __shared__ long long part[4][T / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    StepSums x = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const long long r = __shfl_up(x.rows, d, 64), m = __shfl_up(x.more, d, 64),
                        k = __shfl_up(x.back, d, 64), h = __shfl_up(x.held, d, 64);
        if (lane >= d) x.rows += r, x.more += m, x.back += k, x.held += h;
    }
    if (lane == 63) {
        part[0][wave] = x.rows;
        part[1][wave] = x.more;
        part[2][wave] = x.back;
        part[3][wave] = x.held;
    }
    __syncthreads();
    x.rows -= v.rows, x.more -= v.more, x.back -= v.back;
    total = StepSums();
#pragma unroll
    for (int w = 0; w < T / 64; ++w) {
        const long long r = part[0][w], m = part[1][w], k = part[2][w];
        total.rows += r, total.more += m, total.back += k, total.held += part[3][w];
        if (w < wave) x.rows += r, x.more += m, x.back += k;
    }
    v = x;
}

// The last of n (at least one) ascending numbers that is not above x, the first of which
// is not.
__device__ __forceinline__ int last_not_above(const int *at, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (at[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// the ring's entry k (at most npages) behind entry begin
__device__ __forceinline__ int ring_at(int npages, int begin, int k) {
    const unsigned x = (unsigned)begin + (unsigned)k;
    return (int)(x >= (unsigned)npages ? x - npages : x);
}

// Every workgroup adds up all sequences (they are few numbers, from the caches) and then
// writes its share of the rows, the sequences' entries and the pages given back; so none
// waits for another.  STATE: it also writes the state that the next step starts from,
// which may lie where this step's did: one workgroup, a sequence a thread at most, after all
// have read it.  Several do so if it lies elsewhere; else a second launch does.
//
// A page is taken by the row at its first position: what the list holds from `taken` on
// has no other rows, so each page has one.
template <int T, bool STATE>
__global__ void __launch_bounds__(T) k_kv_step(KvStep a) {
    // where the parts that the sequences are cut into start in the rows, the pages taken
    // and those given back (SUB parts a thread, so that few sequences lie between a part's
    // start and a row's own); the sequences themselves
    constexpr int SUB = STATE ? 1 : 4, PARTS = T * SUB;
    __shared__ int rows_at[PARTS], more_at[PARTS], back_at[PARTS];
    __shared__ StepSeq seq_of[STATE ? T : 1];
    // (of several workgroups half write rows, the others what else there is)
    const int tid = threadIdx.x, wg = blockIdx.x, wgs = gridDim.x;
    const bool do_rows = STATE || blockIdx.y == 0, do_rest = STATE || blockIdx.y == 1;
    const int each = STATE ? 1 : (a.nseq + PARTS - 1) / PARTS;  // sequences of a part
    const int parts = STATE ? a.nseq : a.nseq ? (a.nseq + each - 1) / each : 0;
    const StepRing ring = step_ring(a);
    const int begin = ring.begin, count = ring.count;
    const auto sequence = [&](int i) {
        if constexpr (STATE) return seq_of[i];
        else return step_seq(a, i);
    };
    StepSums part[SUB], at, total;
    for (int j = 0; j < each; ++j)
#pragma unroll
        for (int k = 0; k < SUB; ++k) {
            const int i = (tid * SUB + k) * each + j;
            if (i < a.nseq) {
                const StepSeq s = step_seq(a, i);
                if constexpr (STATE) seq_of[i] = s;
                part[k].add(a, s);
            }
        }
#pragma unroll
    for (int k = 0; k < SUB; ++k) at.add(part[k]);
    step_scan<T>(at, total);
    // (a page is free or in one list: a state whose sum is more than the pool is none that a step
    // left, a page of it would be handed out twice, and ids that go back written over ids that
    // are being taken)
    const bool bad = ring.bad || count + total.held > a.npages;
    const int code =
        (total.rows > a.max_rows ? 1 : 0) | (total.more > count ? 2 : 0) | (bad ? 4 : 0);
    // (a step that succeeds has fewer than 2^31 of each)
#pragma unroll
    for (int k = 0; k < SUB; ++k) {
        rows_at[tid * SUB + k] = (int)at.rows;
        more_at[tid * SUB + k] = (int)at.more;
        back_at[tid * SUB + k] = (int)at.back;
        at.add(part[k]);
    }
    __syncthreads();
    const int nrows = code ? 0 : (int)total.rows, nback = code ? 0 : (int)total.back;
    for (int r = wg * T + tid; do_rows && r < a.max_rows; r += wgs * T) {
        int seq = -1, pos = -1;
        long long slot = -1;
        if (r < nrows) {
            const int c = last_not_above(rows_at, parts, r);
            int row = rows_at[c], more = more_at[c], i = c * each;
            StepSeq s = sequence(i);
            while (r >= row + s.add) {  // within the part: its rows reach past r
                row += s.add;
                more += s.more;
                s = sequence(++i);
            }
            seq = i;
            pos = s.have + r - row;
            const int j = pos >> a.shift, in = pos & ((1 << a.shift) - 1);
            int *const entry = a.pages + (size_t)i * a.max_pages + j;
            int id;
            if (j < s.taken) {
                id = *entry;
            } else {
                id = a.ring[ring_at(a.npages, begin, more + j - s.taken)];
                if (in == 0) *entry = id;
            }
            slot = ((long long)min(max(id, 0), a.npages - 1) << a.shift) | in;
        }
        a.seq[r] = seq;
        a.pos[r] = pos;
        a.slot[r] = slot;
    }
    if (!do_rest) return;
    const int back0 = ring_at(a.npages, begin, count);
    for (int k = wg * T + tid; k < nback; k += wgs * T) {
        const int c = last_not_above(back_at, parts, k);
        int from = back_at[c], i = c * each;
        StepSeq s = sequence(i);
        while (k >= from + step_back(a, s)) {
            from += step_back(a, s);
            s = sequence(++i);
        }
        a.ring[ring_at(a.npages, back0, k)] =
            a.pages[(size_t)i * a.max_pages + step_back_page(a, s, k - from)];
    }
    for (int i = wg * T + tid; i < a.nseq; i += wgs * T) {
        const int c = i / each;
        int rows = rows_at[c], more = more_at[c];
        for (int j = c * each; j < i; ++j) {
            const StepSeq s = sequence(j);
            rows += s.add;
            more += s.more;
        }
        const StepSeq s = sequence(i);
        a.start[i] = code ? 0 : rows;
        a.taken[i] = code ? 0 : more;
        // (of a refused step as given, so that a sequence that was to end still does in the next)
        a.ctx[i] = code ? s.have : s.ended ? 0 : s.have + s.add;
        if (!STATE && apart(a)) step_state(a, i, s, code);
    }
    if (wg == 0 && tid == 0) {
        a.start[a.nseq] = code ? 0 : (int)total.rows;
        a.taken[a.nseq] = code ? 0 : (int)total.more;
        a.status[0] = code;
        a.status[1] = (int)min(total.rows, (long long)INT_MAX);
        a.status[2] = (int)min(total.more, (long long)INT_MAX);
        a.status[3] = nback;
        if (!STATE && apart(a)) ring_state(a, ring, code, total.more, nback);
    }
    if constexpr (STATE) {
        __syncthreads();
        if (tid < a.nseq) step_state(a, tid, seq_of[tid], code);
        if (tid == 0) ring_state(a, ring, code, total.more, nback);
    }
}

// the state after a step of several workgroups, whose status says what it came to
constexpr int STATE_T = 256;
__global__ void __launch_bounds__(STATE_T) k_kv_step_state(KvStep a) {
    const int i = blockIdx.x * STATE_T + threadIdx.x, code = a.status[0];
    if (i < a.nseq) step_state(a, i, step_seq(a, i), code);
    if (i == 0) ring_state(a, step_ring(a), code, a.status[2], a.status[3]);
}

// How many threads (us in a captured graph, 256 threads | 1024 | several workgroups; sequences x
// rows each): 1 x 1 3.3 | 5.6 | 5.9, 64 x 4 4.5 | 6.8 | 6.9, 200 x 1 6.4 | 7.1 | 7.1, 200 x 8
// 11.4 | 8.0 | 7.2, 64 x 1 and 4000 of one 15.8 | 9.0 | 7.0, 1024 x 1 - | 10.8 | 7.8, 1000 x 8
// - | 17.8 | 8.0, 4000 x 2 - | - | 9.6; several whose state lies where it did have a second
// launch, 2 us and the host's.  Of several each has 512 rows or 128 sequences: with twice as
// many 64 x 1 and 4000 take 7.8 and 1000 x 8 8.4, with half 7.0 and 8.0.
void launch_kv_step(const KvStep &a, hipStream_t st) {
    if (a.max_rows <= 2 * STEP_FEW && a.nseq <= STEP_FEW) {
        SI_LAUNCH((k_kv_step<STEP_FEW, true>), dim3(1), dim3(STEP_FEW), 0, st, a);
    } else if (a.max_rows <= 2 * STEP_T && a.nseq <= STEP_T / 2 && !apart(a)) {
        SI_LAUNCH((k_kv_step<STEP_T, true>), dim3(1), dim3(STEP_T), 0, st, a);
    } else {
        const int wgs = std::min(std::max(a.max_rows / 512, a.nseq / 128), 128);
        SI_LAUNCH((k_kv_step<STEP_T, false>), dim3(wgs, 2), dim3(STEP_T), 0, st, a);
        if (!apart(a))
            SI_LAUNCH(k_kv_step_state, dim3(a.nseq / STATE_T + 1), dim3(STATE_T), 0, st, a);
    }
}

// ---------------------------------------------------------------------------
// RoPE and the K/V append by slot (si_rope_kv_append_rows)
//
// The arithmetic and the bits of k_rope_kv: a' = a c - b s, b' = b c + a s, and the fp16
// narrowing.  Memory bounds it: 2060 rows of 28/4 heads of 128 move 73 MB in 14.1 us,
// 5.2 TB/s (large copies 4.9 to 5.9); 40 rows of 14/2 heads of 64 take 3.7 us, the latency of a
// row's place and then its values.  A thread takes four neighbouring pairs of a head (16-byte
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
