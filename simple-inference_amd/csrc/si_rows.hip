// si_rows.hip -- GQA attention of a ragged step's rows over a paged fp16 cache, with a
// sliding window and a few first positions that stay visible (attention_flash,
// attention_kernels.h:80-164, has one query and sees everything).
//
// A row at position p of its sequence sees position t <= p where t > p - window or
// t < sinks.  The (row, head) pairs of a sequence and KV group, row-major, are cut into
// tiles of 32 RT; what a tile's rows see are 32-position tiles of K and V, the sinks' and
// then the window's (RowTile), which a workgroup of RT x KW wavefronts walks: KW of them
// side by side, each met by the RT wavefronts' 32 rows.  Long walks are cut into chunks,
// a workgroup each, whose states (reference, sum, unnormalised output) meet in a second
// kernel.
//
// Per K/V tile a wavefront computes, as the causal prefill kernel does,
//     S^T[pos][row] = K[pos][:] . Q[row][:]          (v_mfma_f32_32x32x16_f16)
//     O^T[d][row] += V^T[d][pos] . P^T[pos][row]
// with Q and P as two fp16 halves each.  A row of q is scaled by a power of two to 2^14,
// fac takes it back: a weight is 2^(fac s - c + 11), c a reference near the scores of the
// tile at hand: it moves when the tile's largest lies more than 2^4 over it, or 2^12
// under.  So a weight is off by at most 2^-23 of itself and 2^-24 of its tile's largest,
// also behind a position that outweighs the rest (an attention sink, whose values are
// small): sums in 32 bits hold both.  The sinks' tiles
// have no other positions in them (a window's tile that they share is met twice).
//
// Where a mask cuts a tile its hidden scores are replaced (not added to), and V's values
// there are looked at: 0 x infinity would be NaN.  Only if one is not finite, the rows
// that see it are marked by NaN, and the tile in LDS has zeros in such places from then on.
//
// What a row sees of infinities and NaN it gets as the definition has it, wherever they lie: a score
// of NaN or +inf makes its outputs NaN, one of -inf has no weight, and an infinity of V stays
// one.  Two halves of q or of a weight would make NaN of them, or the lo half's sign; so a
// workgroup whose outputs are not finite walks again (rows_walk, SURE), a tile at a time: a call
// whose workgroups all do takes three to four times as long (64 x 4096 91 -> 284 us, a prompt of
// 8000 404 -> 1700).  Where none does it costs an instruction an output and a barrier (us, without
// | with: a piece of 333 rows 26.4 | 26.9, pieces among tokens 96.5 | 97.4, a prompt of 8000 404 |
// 404, 64 x 4096 90.6 | 90.7).
//
// What bounds it (MI355X; a plain read reaches 6.2 TB/s, a large f16 product 1.18 PFLOP/s):
//   single tokens, 64 sequences in windows of 4096, 28/4 heads of 128: memory, 539 MB in
//     88 to 90 us, 6.1 TB/s.
//   few of them (2 x 65536 positions of 12/2 heads, 16 x 4096 of 28/4 with up to 8 rows): the
//     chunks' start, 129 MB in 24 us and 92 MB in 29 us, and the merge's launch after them, 4.5.
//   one short window (1024 of 14/2 heads of 64): latency, 6.3 us + 3.0 of the merge.
//   prompts (8000 rows in a window of 2048, 28/4): 415 us, 205 GFLOP, twice that issued for the
//     halves: 1.0 PFLOP/s at the 1.9 GHz that the clock keeps.  Matrix cores busy half of the
//     cycles; without the lo halves 300 us (and errors of 2^-11), without exponentials 366.
//   pieces of prompts (333 rows after 1500) and pieces among single tokens: 26 and 97 to 107 us, the
//     latency of the steps and of a workgroup's start (6 us: its sequence, pages, q).
// Why these tiles: a lane holds one row's half of a tile's scores, so that a row's maximum and sum
// take one exchange and its weights are the next product's operand as they are, without LDS.  One
// 32-row tile a workgroup leaves a wavefront its own K/V tiles and no barrier; with four a staged
// tile is read from LDS by four wavefronts and from memory once.
#include <limits.h>
#include <algorithm>

#include "si_device.hpp"
#include "si_kernels.hpp"
#include "si_tiles.hpp"

namespace si {

constexpr float RW_UP = 11.0f;    // log2 of a weight's unit
constexpr float RW_OVER = 4.0f;   // how far a tile's largest may lie over the reference
constexpr float RW_UNDER = 12.0f; // and under it
constexpr float RW_ROOM = 100.0f; // log2 of a sum's largest value (times V's, 2^16)

// ---------------------------------------------------------------------------
// What a tile's rows see
// ---------------------------------------------------------------------------
struct RowTile {
    int seq, row0;      // the sequence; its first row in q (row0 + t / per is pair t's)
    int p0;             // position of row0
    int pair0, pairs;   // the tile's (row, head) pairs of this KV group
    int first, last;    // positions of the first and the last of them
    int sink_tiles, w0; // K/V tiles of the sinks; the window's first one
    int ntiles;         // of both
    // the v-th of them
    __device__ __forceinline__ int tile(int v) const {
        return v < sink_tiles ? v : w0 + v - sink_tiles;
    }
    // whether rows at positions p0 to p1 see anything of the v-th, and all of it (of a
    // sinks' tile the sinks, of a window's tile the others)
    __device__ __forceinline__ bool touches(const RowsArgs &a, int v, int p0, int p1) const {
        const int kv0 = tile(v) * PF_T;
        return kv0 <= p1 && (v < sink_tiles || kv0 + PF_T - 1 > p0 - a.window);
    }
    __device__ __forceinline__ bool inside(const RowsArgs &a, int v, int p0, int p1) const {
        const int kv0 = tile(v) * PF_T;
        return kv0 + PF_T - 1 <= p0 && (v < sink_tiles ? kv0 + PF_T <= a.sinks
                                                       : kv0 >= a.sinks && kv0 > p1 - a.window);
    }
};

// rows of sequence i within the call's limits, the first and its position
__device__ __forceinline__ int seq_rows(const RowsArgs &a, int i, int &row0, int &p0) {
    const int s0 = max(a.start[i], 0), s1 = max(a.start[i + 1], 0);
    row0 = min(s0, a.max_rows);
    // (a context below 0 is 0, of which the starts' difference may be taken in 32 bits; rows are
    // fewer than 2^24: what lies further before position 0 is all hidden)
    p0 = max(min(max(a.ctx[i], 0), a.max_ctx) - (s1 - s0), -(1 << 24));
    return min(max(min(s1, a.max_rows) - row0, 0), a.max_new);
}

__device__ __forceinline__ void row_tile(const RowsArgs &a, int tile_rows, int i, int k,
                                         RowTile &t) {
    const int per = a.qheads / a.kvheads;
    const int n = seq_rows(a, i, t.row0, t.p0);
    t.seq = i;
    t.pair0 = k * tile_rows;
    t.pairs = min(n * per - t.pair0, tile_rows);
    if (t.pairs <= 0) {
        t.pairs = t.ntiles = 0;
        return;
    }
    t.first = t.p0 + t.pair0 / per;
    t.last = t.p0 + (t.pair0 + t.pairs - 1) / per;
    const int from = max(t.first - a.window + 1, a.sinks);
    t.w0 = from / PF_T;
    t.sink_tiles = min((a.sinks + PF_T - 1) / PF_T, t.last < 0 ? 0 : t.last / PF_T + 1);
    t.ntiles = t.sink_tiles + (t.last < from ? 0 : t.last / PF_T - t.w0 + 1);
}

// Tile number `tile` of the call: one a sequence (ONE: max_new rows fill no more), or the
// sequences' tiles one after another, the last first (a prompt's last rows see most), found
// by a prefix sum over the sequences.  Every thread of the workgroup; false past the last.
template <bool ONE, int NT>
__device__ __forceinline__ bool find_tile(const RowsArgs &a, int tile_rows, int tile, RowTile &t) {
    if constexpr (ONE) {
        row_tile(a, tile_rows, tile, 0, t);
        return t.pairs > 0;
    } else {
        // (64 bits: starts that are no prefix sums may give every sequence all rows)
        __shared__ long long red[NT / 64];
        __shared__ int found[2];
        const int per = a.qheads / a.kvheads, tid = threadIdx.x;
        const auto tiles = [&](int i) {
            int r, p;
            return (seq_rows(a, i, r, p) * per + tile_rows - 1) / tile_rows;
        };
        if (a.nseq == 1) {  // (its tiles are the call's)
            const int k = tiles(0) - 1 - tile;
            if (k < 0) return false;
            row_tile(a, tile_rows, 0, k, t);
            return true;
        }
        const int each = (a.nseq + NT - 1) / NT;
        const int i0 = min(tid * each, a.nseq), i1 = min(i0 + each, a.nseq);
        long long sum = 0;
        for (int i = i0; i < i1; ++i) sum += tiles(i);
        long long x = sum;
        for (int d = 1; d < 64; d <<= 1) {
            const long long y = __shfl_up(x, d, 64);
            if ((tid & 63) >= d) x += y;
        }
        if ((tid & 63) == 63) red[tid >> 6] = x;
        __syncthreads();
        long long base = x - sum, total = 0;
        for (int w = 0; w < NT / 64; ++w) {
            if (w < (tid >> 6)) base += red[w];
            total += red[w];
        }
        const long long at = total - 1 - tile;
        if (at < 0) return false;
        if (at >= base && at < base + sum)  // (one thread's)
            for (int i = i0; i < i1; ++i) {
                const int n = tiles(i);
                if (at < base + n) {
                    found[0] = i;
                    found[1] = (int)(at - base);
                    break;
                }
                base += n;
            }
        __syncthreads();
        row_tile(a, tile_rows, __builtin_amdgcn_readfirstlane(found[0]),
                 __builtin_amdgcn_readfirstlane(found[1]), t);
        return true;
    }
}

// ---------------------------------------------------------------------------
// The chunks' states in the workspace: [tile][KV group][chunk] blocks of rows x D outputs,
// then as many rows x (reference, sum)
// ---------------------------------------------------------------------------
struct RowsParts {
    float *o, *m;
    int rows;  // rows of a block that may be used
    int chunks, chunk_tiles;
};

__device__ __forceinline__ size_t part_row(const RowsParts &pt, int kvheads, int tile, int g,
                                           int chunk, int row) {
    return (((size_t)tile * kvheads + g) * pt.chunks + chunk) * pt.rows + row;
}

// 4 values of a row's head (8 lanes hold a Q8_0 block), zeros before position 0
template <int D>
__device__ __forceinline__ void rows_store(const RowsArgs &a, int row, int head, int dd, int pos,
                                           float (&y)[4]) {
    if (pos < 0)
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = 0.0f;
    const size_t off = ((size_t)row * a.qheads + head) * D + dd;
    *(f4 *)(a.attn + off) = (f4){y[0], y[1], y[2], y[3]};
    if (!a.qs) return;
    uint16_t dbits;
    int sum;
    *(uint32_t *)(a.qs + off) = quant_block_oct(y, dbits, sum);
    if ((threadIdx.x & 7) == 0) {
        a.d[off / SI_QK] = dbits;
        if (a.bsum) a.bsum[off / SI_QK] = (int16_t)sum;
    }
}

__device__ __forceinline__ bool finite_h(_Float16 x) {
    return (__builtin_bit_cast(uint16_t, x) & 0x7c00u) != 0x7c00u;
}
// A state's factor, 2^-149 where it would be 0 in 32 bits, so that an infinity among the state's
// outputs stays one (a finite output is moved by less than the 0 below 2^-126 moves it)
__device__ __forceinline__ float some(float f) { return f < 0x1p-149f ? 0x1p-149f : f; }

// AHEAD: steps that a stage's copies are issued before their use (RT > 1).
template <int D, int RT, int KW, int AHEAD>
struct RowsForm {
    static constexpr int NWV = RT * KW, NT = NWV * 64, TB = PF_T * D * 2;  // bytes of a K (V) tile
    static constexpr int OROW = D + PF_OPAD;
    // RT > 1: AHEAD + 1 stages (K tiles, then V tiles) used in turn, one barrier per step.
    // RT == 1: each wavefront stages its own tiles, K in sb and V in sb1, both refilled as
    // soon as they are in registers (no barrier).  KW > 1: at the end the wavefronts'
    // outputs, where there are two arrays half of them in each.
    static constexpr bool DB = RT > 1;
    static constexpr int STAGE = (DB ? 2 : 1) * KW * TB, NSTAGE = DB ? AHEAD + 1 : 1;
    static constexpr int MRG_W = DB ? NWV : (NWV + 1) / 2;
    static constexpr int MRG = KW > 1 ? MRG_W * PF_T * OROW * 4 : 0;
    static constexpr int SB = NSTAGE * STAGE > MRG ? NSTAGE * STAGE : MRG;
};

// A workgroup's share of the call: a KV group's tile of rows, and a chunk of its tiles of K and V,
// from v0 to v1
struct RowsShare {
    RowTile rw;
    int g, tile, chunk, v0, v1;
};

// A wavefront's rows, and lane t's own of them
struct RowsWave {
    int kw, rt, lane, t, hh;
    bool any;                 // whether there are some
    int first, last;          // positions of the first and the last
    int row, head, pos;       // lane t's (the last one again past it)
    template <int RT>
    static __device__ __forceinline__ RowsWave of(const RowsArgs &a, const RowsShare &sh, int tid) {
        RowsWave w;
        const RowTile &rw = sh.rw;
        const int per = a.qheads / a.kvheads, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        w.lane = tid & 63;
        w.kw = wave / RT, w.rt = wave % RT;
        w.t = w.lane & 31, w.hh = w.lane >> 5;
        const int p0 = rw.pair0 + min(32 * w.rt, rw.pairs - 1);
        const int p1 = rw.pair0 + min(32 * w.rt + 31, rw.pairs - 1);
        w.any = 32 * w.rt < rw.pairs;
        w.first = rw.p0 + p0 / per, w.last = rw.p0 + p1 / per;
        const int pair = min(rw.pair0 + 32 * w.rt + w.t, p1);
        w.row = rw.row0 + pair / per, w.head = sh.g * per + pair % per;
        w.pos = rw.p0 + pair / per;
        return w;
    }
};

// One wavefront's walk over its tiles: row t's reference c, this lane's share of the sum, and the
// outputs (lane (t, hh): O[row t][32 dt + 8 (r / 4) + 4 hh + r % 4] in o[dt][r]).
//
// An infinity or NaN that a row sees, in K or V, makes its sums NaN, or infinite by the sign of a
// lo half (q's and the weights' are of either sign, or 0).  A workgroup with such outputs walks
// again, with SURE, a tile at a time: scores that are not finite from q's hi halves alone, whose
// signs are q's; V's infinities and NaN, with zeros in their places, counted apart by what rows
// see them.
//
// PAGE: pages of 32 positions and more, whole tiles (32), of 16 where an instruction's rows are
// whole (16: two a tile), of any (1: each lane looks up its own row's: with 1 in place of 32, us,
// 64 x 4096 of 28/4 heads of 128 102 | 91, 8000 rows of 2048 448 | 415, a piece of 333 rows 33 | 25;
// in place of 16, 1024 positions of 14/2 of 64 10.5 | 9.6).
template <int D, int RT, int KW, int AHEAD, bool ONE, int PAGE, bool SURE>
__device__ __forceinline__ void rows_walk(const RowsArgs &a, const RowsShare &sh, int tid,
                                          uint8_t *sb, uint8_t *sb1, int *bad_step, float &c,
                                          float &lsum, f16v (&o)[D / 32]) {
    using F = RowsForm<D, RT, KW, AHEAD>;
    constexpr int KS = D / 16, DT = D / 32, CH = D / 8, TB = F::TB;
    constexpr int TI = TB / 1024;            // copy instructions per tile
    constexpr int TIW = (TI + RT - 1) / RT;  // of one wavefront
    constexpr bool DB = F::DB;
    constexpr int STAGE = F::STAGE, NSTAGE = F::NSTAGE;
    // (K and V that one workgroup reads are kept out of the caches: us, 64 x 4096 of 28/4 heads
    // 98 | 91, 2 x 65536 of 12/2 32 | 29; a prompt's are read by many)
    constexpr int AUX = ONE ? 2 : 0;
    const RowTile &rw = sh.rw;
    const int g = sh.g, v0 = sh.v0, v1 = sh.v1, kvd = a.kvheads * D;
    const int steps = (v1 - v0 + KW - 1) / KW;
    const RowsWave me = RowsWave::of<RT>(a, sh, tid);
    const int lane = me.lane, kw = me.kw, rt = me.rt, t = me.t, hh = me.hh;
    const int wfirst = me.first, wlast = me.last, prow = me.pos;
    const bool rows_here = me.any;

    // lane (t, hh) has k-slice hh of row t of q: on its way while the pages are looked up
    float4 x0[KS], x1[KS];
    {
        const float *qrow = a.q + ((size_t)me.row * a.qheads + me.head) * D + 8 * hh;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            x0[ks] = *(const float4 *)(qrow + 16 * ks);
            x1[ks] = *(const float4 *)(qrow + 16 * ks + 4);
        }
    }
    // this wavefront's copies of a tile: instruction i takes the 16-byte units
    // 64 n .. 64 n + 63 of the tile (LDS order), n = rt + RT i.  Where these are whole rows
    // (RPI of them) the lane's offset within them is one number for V, and for K one that
    // an XOR turns into each instruction's (a row's bytes are a multiple of its D 2).
    constexpr bool WHOLE = 64 % CH == 0;
    constexpr int RPI = WHOLE ? 64 / CH : 1;
    const int lrow = lane / CH, lslot = lane % CH;
    const int kcol = pf_k_chunk<D>(lrow, lslot) * 16, vcol = pf_v_slot<D>(lrow, lslot) * 16;
    // row of the lane's unit of instruction i within the tile, and its bytes from the row's start
    const auto unit = [&](int i, bool is_k, int &row, int &col) {
        const int n = rt + RT * i;
        if constexpr (WHOLE) {
            row = RPI * n + lrow;
            col = is_k ? kcol ^ (pf_k_slot<D>(RPI * n, 0) * 16) : vcol;
        } else {
            const int p = n * 64 + lane;
            row = p / CH;
            col = (is_k ? pf_k_chunk<D>(row, p % CH) : pf_v_slot<D>(row, p % CH)) * 16;
        }
    };
    // the pages of a step's tile (past the chunk: its last one again): of its first
    // position, of the one 16 behind it too, or of position t
    // (read as constant data: through the scalar cache, whose loads are not among those
    // that the waits for copies count)
    typedef const __attribute__((address_space(4))) int const_int;
    const const_int *list = (const const_int *)(a.pg.pages + (size_t)rw.seq * a.pg.max_pages);
    struct Pages {
        int id, second;
    };
    const auto nth = [&](int st) { return min(v0 + st * KW + kw, v1 - 1); };
    const auto id_of = [&](int pos) {
        const int id = list[min(pos >> a.pg.shift, a.pg.max_pages - 1)];
        return min(max(id, 0), a.pg.npages - 1);
    };
    const auto page_of = [&](int st) {
        const int pos = rw.tile(nth(st)) * PF_T;
        return Pages{id_of(PAGE == 1 ? pos + t : pos), PAGE == 16 ? id_of(pos + 16) : 0};
    };
    const auto copy = [&](const uint16_t *pool, uint8_t *dst, int st, Pages page, bool is_k) {
        const int pos0 = rw.tile(nth(st)) * PF_T, mask = (1 << a.pg.shift) - 1;
        uint8_t *const to = dst + kw * TB + 1024 * rt;
        if constexpr (PAGE > 1) {
            const auto at = [&](int id, int pos) {
                const size_t row0 = ((size_t)__builtin_amdgcn_readfirstlane(id) << a.pg.shift) |
                                    (size_t)(pos & mask);
                return buf_rsrc(pool + row0 * kvd + g * D, 0x7fffffffu);
            };
            const __amdgpu_buffer_rsrc_t rs = at(page.id, pos0);
            const __amdgpu_buffer_rsrc_t rs2 = PAGE == 16 ? at(page.second, pos0 + 16) : rs;
#pragma unroll
            for (int i = 0; i < TIW; ++i)
                if (TI % RT == 0 || rt + RT * i < TI) {
                    if constexpr (WHOLE) {
                        const int row = RPI * (rt + RT * i);  // the instruction's first
                        const int x = is_k ? pf_k_slot<D>(row, 0) * 16 : 0;
                        const bool second = PAGE == 16 && row >= 16;  // wavefront-uniform
                        lds_copy16<AUX>(second ? rs2 : rs, to + 1024 * RT * i,
                                        (uint32_t)(lrow * (kvd * 2) + ((is_k ? kcol : vcol) ^ x)),
                                        (second ? row - 16 : row) * (kvd * 2));
                    } else {
                        int row, col;
                        unit(i, is_k, row, col);
                        lds_copy16<AUX>(rs, to + 1024 * RT * i,
                                        (uint32_t)(row * (kvd * 2) + col), 0);
                    }
                }
        } else {
#pragma unroll
            for (int i = 0; i < TIW; ++i)
                if (TI % RT == 0 || rt + RT * i < TI) {
                    int r, col;
                    unit(i, is_k, r, col);
                    const int id = __shfl(page.id, r, 64);
                    const size_t row = ((size_t)id << a.pg.shift) | (size_t)((pos0 + r) & mask);
                    lds_copy16_at((const uint8_t *)(pool + row * kvd + g * D) + col,
                                  to + 1024 * RT * i);
                }
        }
    };
    // the first copies: K up to step AHEAD and V one step less (RT == 1: of step 0)
    Pages page = {}, page1 = {};
    if (!SURE && steps > 0) {
        page = page_of(0);
        copy(a.k, sb, 0, page, true);
        if constexpr (DB) {
#pragma unroll
            for (int s = 0; s < AHEAD; ++s) {
                if (s < steps) copy(a.v, sb + s * STAGE + KW * TB, s, page, false);
                page = page_of(s + 1);
                if (s + 1 < steps) copy(a.k, sb + (s + 1) * STAGE, s + 1, page, true);
            }
            page1 = page;
            page = page_of(AHEAD + 1);
        } else {
            copy(a.v, sb1, 0, page, false);
            page = page_of(1);
        }
    }

    // Q^T as the B operand of the score MFMA (columns past the last row repeat it and are
    // never stored)
    h8 qh[KS], ql[KS];
    float fac;
    {
        float big = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
            big = fmaxf(big, fmaxf(fmaxf(fmaxf(fabsf(x0[ks].x), fabsf(x0[ks].y)),
                                         fmaxf(fabsf(x0[ks].z), fabsf(x0[ks].w))),
                                   fmaxf(fmaxf(fabsf(x1[ks].x), fabsf(x1[ks].y)),
                                         fmaxf(fabsf(x1[ks].z), fabsf(x1[ks].w)))));
        big = fmaxf(big, swap32_f(big));
        // the row's largest value to 2^14 (one below 2^-60 makes no score)
        const int up = 14 - max((int)(f2u(big) >> 23) - 127, -60);
        // (past 2^80 a weight is 0 or 1 either way, and a score, 2^38 at most, times it finite)
        fac = fminf(__builtin_amdgcn_ldexpf(a.scale2, -up), 0x1p80f);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            float x[8] = {x0[ks].x, x0[ks].y, x0[ks].z, x0[ks].w,
                          x1[ks].x, x1[ks].y, x1[ks].z, x1[ks].w};
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = __builtin_amdgcn_ldexpf(x[e], up);
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                pf_h2 hi, lo;
                split_pair(x[e], x[e + 1], hi, lo);
                qh[ks][e] = hi[0];
                qh[ks][e + 1] = hi[1];
                ql[ks][e] = lo[0];
                ql[ks][e + 1] = lo[1];
            }
        }
    }

    // operand addresses within a stage: K row t, chunk 2 ks + hh; V rows
    // 16 s2 + 8 e + 4 hh + s / 4 (s = lane % 16), columns 32 dt + 16 (lane / 16 % 2) +
    // 4 (s % 4), as the transposing read takes them
    const int s16 = lane & 15;
    int ka[KS], va[DT];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
        ka[ks] = kw * TB + t * D * 2 + pf_k_slot<D>(t, 2 * ks + hh) * 16;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
        va[dt] = kw * TB + (4 * hh + (s16 >> 2)) * D * 2 +
                 pf_v_slot<D>(s16 >> 2, 4 * dt + 2 * ((lane >> 4) & 1) + ((s16 & 3) >> 1)) * 16 +
                 (s16 & 1) * 8;

    c = -INFINITY;
    lsum = 0.0f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = (f16v){};

    const auto products = [&](const h8 (&x)[KS]) {
        // the lo products first: they round at their own small magnitude
        f16v s = (f16v){};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[ks], ql[ks], s, 0, 0, 0);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[ks], qh[ks], s, 0, 0, 0);
        return s;
    };
    const auto scores = [&](const uint8_t *kt) {
        h8 x[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) x[ks] = *(const h8 *)(kt + ka[ks]);
        return products(x);
    };
    // the positions of the v-th tile that lane t's row sees: those from `from` on, `width`
    // more, counted from the lane's first, kv0 + 4 hh (register r: 8 (r / 4) + r % 4 behind it)
    struct Seen {
        int from, width;
        __device__ __forceinline__ bool at(int r) const {
            return (unsigned)(8 * (r >> 2) + (r & 3) - from) <= (unsigned)width;
        }
    };
    const auto seen_of = [&](int v) {
        const bool sink = v < rw.sink_tiles;
        const int lo = sink ? 0 : max(prow - a.window + 1, a.sinks);
        const int hi = sink ? min(prow, a.sinks - 1) : prow;
        const int at = rw.tile(v) * PF_T + 4 * hh;
        return hi < lo ? Seen{64, 0} : Seen{lo - at, hi - lo};
    };
    h8 ph[2], pl[2];  // the tile's weights
    float one = 1.0f;
    asm("" : "+s"(one));
    const auto refer = [&](f16v &s, int v, bool cut) {
        if (cut) {  // wavefront-uniform
            const Seen seen = seen_of(v);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = seen.at(r) ? s[r] : -INFINITY;
        }
        // (a plain operation reads the matrix results first: the compiler puts the wait
        // states they need before it, which it would not before the inline instructions
        // that follow from it)
        float mx = fmaxf(s[0], s[1]);
#pragma unroll
        for (int r = 2; r < 16; r += 2) mx = max3_f(mx, s[r], s[r + 1]);
        mx = fmaxf(mx, swap32_f(mx)) * fac;
        const float d = mx - c;
        if (__ballot((d > RW_OVER) | (d < -RW_UNDER))) {
            // up to the tile's largest; or down to it, as far as the sums have room
            // (both halves of a row take the same step)
            const float l = fmaxf(lsum, swap32_f(lsum));
            const float room = RW_ROOM - (float)((int)(f2u(l) >> 23) - 127);
            float to = c;
            if (d > RW_OVER) to = mx;
            else if (d < -RW_UNDER && mx > -INFINITY) to = c - fminf(-d, fmaxf(room, 0.0f));
            const float alpha = to == c ? 1.0f : some(__builtin_amdgcn_exp2f(c - to));
            c = to;
            lsum *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
        }
    };
    const auto weights = [&](const f16v &s) {
        const float up = RW_UP - (c == -INFINITY ? 0.0f : c);
        float ps = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
            const float p0 = __builtin_amdgcn_exp2f(fmaf(s[r], fac, up));
            const float p1 = __builtin_amdgcn_exp2f(fmaf(s[r + 1], fac, up));
            ps += p0;
            ps += p1;
            const pf_h2 hi = __builtin_convertvector((pf_f2){p0, p1}, pf_h2);
            ph[r >> 3][r & 7] = hi[0];
            ph[r >> 3][(r & 7) + 1] = hi[1];
            // (a mixed-precision fma each, as the factor 1 is not the compiler's to see)
            pl[r >> 3][r & 7] = (_Float16)fmaf(-(float)hi[0], one, p0);
            pl[r >> 3][(r & 7) + 1] = (_Float16)fmaf(-(float)hi[1], one, p1);
        }
        lsum += ps;
    };
    // k-step s2 covers positions 16 s2 + 8 (e / 4) + 4 hh + e % 4 (e = element 0..7), the
    // positions of registers 8 s2 + e of the score output
    const auto v_operand = [&](const uint8_t *vt, int dt, int s2) {
        const h4 x0 = __builtin_bit_cast(h4, lds_read_tr16(vt + va[dt] + 16 * s2 * D * 2));
        const h4 x1 = __builtin_bit_cast(h4, lds_read_tr16(vt + va[dt] + (16 * s2 + 8) * D * 2));
        return (h8){x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
    };
    // The scores of K tile kt among the weights of s, and V's operands on their way: the
    // matrix cores and the vector ALU work side by side, each product followed by its share
    // of the weights (the order as written: left to itself the compiler puts the products
    // together).
    const auto scores_and_weights = [&](const uint8_t *kt, const f16v &s, const uint8_t *vt) {
        constexpr int SLOTS = 2 * KS;
        const float up = RW_UP - (c == -INFINITY ? 0.0f : c);
        f16v n = (f16v){};
        h8 x[KS], vx[2 * DT];
        float p[16], ps = 0.0f;
        x[0] = *(const h8 *)(kt + ka[0]);
        x[1] = *(const h8 *)(kt + ka[1]);
#pragma unroll
        for (int i = 0; i < SLOTS; ++i) {
            const int ks = i / 2;
            if (i % 2 == 0 && ks + 2 < KS) x[ks + 2] = *(const h8 *)(kt + ka[ks + 2]);
            n = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[ks], i % 2 ? qh[ks] : ql[ks], n, 0, 0, 0);
#pragma unroll
            for (int r = i * 16 / SLOTS; r < (i + 1) * 16 / SLOTS; ++r) {
                p[r] = __builtin_amdgcn_exp2f(fmaf(s[r], fac, up));
                if (r >= 2) {  // (the exponential before the last is done)
                    const int e = r - 2;
                    ps += p[e];
                    ph[e >> 3][e & 7] = (_Float16)p[e];
                    pl[e >> 3][e & 7] = (_Float16)fmaf(-(float)ph[e >> 3][e & 7], one, p[e]);
                }
            }
            // (the first positions' operands in the last slots; registers are short)
#pragma unroll
            for (int k = 0; k < DT; ++k)
                if (i == SLOTS - DT + k) vx[2 * k] = v_operand(vt, k, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int e = 14; e < 16; ++e) {
            ps += p[e];
            ph[1][e & 7] = (_Float16)p[e];
            pl[1][e & 7] = (_Float16)fmaf(-(float)ph[1][e & 7], one, p[e]);
        }
        lsum += ps;
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                if (s2 == 0) vx[2 * dt + 1] = v_operand(vt, dt, 1);
                const h8 y = vx[2 * dt + s2];
                o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(y, ph[s2], o[dt], 0, 0, 0);
                o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(y, pl[s2], o[dt], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
        return n;
    };
    // whether this wavefront's share of a V tile holds an infinity or NaN (exponents of all
    // ones)
    typedef uint32_t w4 __attribute__((ext_vector_type(4)));
    const auto any_bad = [&](const uint8_t *vt) {
        uint32_t bad = 0;
#pragma unroll
        for (int i = 0; i < TIW; ++i)
            if (TI % RT == 0 || rt + RT * i < TI) {
                const w4 w = *(const w4 *)(vt + kw * TB + 1024 * (rt + RT * i) + 16 * lane);
#pragma unroll
                for (int e = 0; e < 4; ++e) bad |= (w[e] & 0x7c007c00u) + 0x04000400u;
            }
        return __ballot((bad & 0x80008000u) != 0) != 0;
    };
    // what rows see such values: NaN for the time being (the walk is taken again for them)
    const auto mark_bad = [&](const uint8_t *vt, int v) {
        h8 seen[2];
        const Seen sn = seen_of(v);
#pragma unroll
        for (int r = 0; r < 16; ++r)
            seen[r >> 3][r & 7] = sn.at(r) ? (_Float16)1.0f : (_Float16)0.0f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            f16v n = (f16v){};
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2) {
                h8 k = v_operand(vt, dt, s2);
#pragma unroll
                for (int e = 0; e < 8; ++e) k[e] = (_Float16)(finite_h(k[e]) ? 0.0f : 1.0f);
                n = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, seen[s2], n, 0, 0, 0);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) o[dt][e] = n[e] > 0.0f ? __builtin_nanf("") : o[dt][e];
        }
    };
    // this wavefront's share of a V tile with zeros in their places
    const auto drop_bad = [&](uint8_t *vt) {
#pragma unroll
        for (int i = 0; i < TIW; ++i)
            if (TI % RT == 0 || rt + RT * i < TI) {
                w4 *at = (w4 *)(vt + kw * TB + 1024 * (rt + RT * i) + 16 * lane);
                w4 w = *at;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t bad = (((w[e] & 0x7c007c00u) + 0x04000400u) >> 15) & 0x10001u;
                    w[e] &= ~(bad * 0xffffu);
                }
                *at = w;
            }
    };
    if constexpr (SURE) {
        uint8_t *const vt = DB ? sb + KW * TB : sb1;
        bool in_turn = false;
#pragma unroll 1
        for (int st = 0; st < steps; ++st) {
            pf_wait<0>();  // the last tile is read
            if constexpr (DB) pf_barrier();
            const Pages now = page_of(st);
            copy(a.k, sb, st, now, true);
            copy(a.v, vt, st, now, false);
            pf_wait<0>();
            if constexpr (DB) pf_barrier();
            const int v = nth(st);
            if (!(v0 + st * KW + kw < v1 && rows_here && rw.touches(a, v, wfirst, wlast))) {
                in_turn = false;
                continue;  // (wavefront-uniform; the barriers are at the loop's head)
            }
            // The first walk's sums in its order, so that rows without such values keep their
            // bits: there, after a step that computed weights, q's halves take turns.  (A load,
            // its products, the next: registers are short.)
            f16v s = (f16v){}, by_hi = (f16v){};
            const auto product = [&](int ks, bool hi) {
                const h8 x = *(const h8 *)(sb + ka[ks]);
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, hi ? qh[ks] : ql[ks], s, 0, 0, 0);
                if (hi) by_hi = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, qh[ks], by_hi, 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            };
            if (in_turn) {
#pragma unroll
                for (int i = 0; i < 2 * KS; ++i) product(i / 2, i % 2);
            } else {
#pragma unroll
                for (int i = 0; i < 2 * KS; ++i) product(i % KS, i >= KS);
            }
            in_turn = DB;
#pragma unroll
            for (int r = 0; r < 16; ++r)
                s[r] = fabsf(s[r]) < __builtin_inff() ? s[r] : by_hi[r];
            refer(s, v, true);
            weights(s);
            // positions of any weight, and visible ones of none (a score of -inf), a bit each
            uint32_t live = 0, none = 0;
            {
                const Seen sn = seen_of(v);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    if (sn.at(r) && s[r] != -INFINITY) live |= 1u << r;
                    if (sn.at(r) && s[r] == -INFINITY) none |= 1u << r;
                }
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                // infinities count 1, negative ones 64, NaN and products with 0 both (exactly: a
                // tile has 32 positions)
                f16v n = (f16v){};
#pragma unroll
                for (int s2 = 0; s2 < 2; ++s2) {
                    const h8 y = v_operand(vt, dt, s2);
                    h8 x, w;
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = finite_h(y[e]) ? y[e] : (_Float16)0.0f;
                    o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, ph[s2], o[dt], 0, 0, 0);
                    o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, pl[s2], o[dt], 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint16_t b = __builtin_bit_cast(uint16_t, (_Float16)y[e]);
                        const float kind = (b & 0x3ffu) ? 65.0f : b >> 15 ? 64.0f : 1.0f;
                        x[e] = (_Float16)(finite_h(y[e]) ? 0.0f : kind);
                        w[e] = (_Float16)(float)((live >> (8 * s2 + e)) & 1u);
                    }
                    n = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, w, n, 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        x[e] = (_Float16)(finite_h(y[e]) ? 0.0f : 65.0f);
                        w[e] = (_Float16)(float)((none >> (8 * s2 + e)) & 1u);
                    }
                    n = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, w, n, 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int k = (int)n[e];
                    const float up = (k & 63) ? __builtin_inff() : 0.0f;
                    const float down = (k >> 6) ? -__builtin_inff() : 0.0f;
                    o[dt][e] += up + down;
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    } else if constexpr (DB) {
        // K runs a step ahead of V: a step's weights are computed among the next one's
        // scores.  After its barrier the next K and this V are in, and the buffers of the
        // last K and V free; the copies into them have AHEAD steps to arrive.
        if (tid < 2) bad_step[tid] = 0;
        pf_wait<0>();
        pf_barrier();
        f16v s0 = (f16v){}, s1 = (f16v){};
        if (steps > 0) s0 = scores(sb);
        int at = 0;  // st % NSTAGE
        const auto step = [&](f16v &s, f16v &next, int st) {
            const int after = at + 1 == NSTAGE ? 0 : at + 1, before = at ? at - 1 : NSTAGE - 1;
            uint8_t *const cur = sb + at * STAGE, *const nxt = sb + after * STAGE;
            // (copies of the steps since may be on their way; D of 96: fewer for some)
            if (st + AHEAD < steps) pf_wait<(AHEAD - 1) * 2 * (TI / RT)>();
            else pf_wait<0>();
            pf_barrier();
            // (the next page's load before the copies: a wait for it is none for them)
            const Pages page2 = page_of(st + AHEAD + 2);
            asm volatile("" ::: "memory");
            if (st + AHEAD < steps)
                copy(a.v, sb + before * STAGE + KW * TB, st + AHEAD, page1, false);
            if (st + AHEAD + 1 < steps) copy(a.k, cur, st + AHEAD + 1, page, true);
            page1 = page;
            page = page2;
            at = after;
            const int v = nth(st);
            const bool use = v0 + st * KW + kw < v1 && rows_here &&
                             rw.touches(a, v, wfirst, wlast);  // wavefront-uniform
            uint8_t *const vt = cur + KW * TB;
            // a step with a tile that some row of the workgroup sees in part
            bool cut = false;
#pragma unroll
            for (int k = 0; k < KW; ++k)
                cut |= !rw.inside(a, min(v0 + st * KW + k, v1 - 1), rw.first, rw.last);
            if (use) refer(s, v, cut && !rw.inside(a, v, wfirst, wlast));
            if (cut) {  // workgroup-uniform
                if (any_bad(vt) && lane == 0) bad_step[st & 1] = 1;
                __syncthreads();
                if (bad_step[st & 1]) {
                    if (use) mark_bad(vt, v);
                    __syncthreads();
                    drop_bad(vt);
                    __syncthreads();
                    if (tid == 0) bad_step[st & 1] = 0;  // (next set two barriers from here)
                }
            }
            // (past the last step the next scores are of no use)
            if (use) {
                next = scores_and_weights(nxt, s, vt);
            } else if (rows_here) {
                next = scores(nxt);
            }
        };
        for (int st = 0; st < steps; st += 2) {
            step(s0, s1, st);
            if (st + 1 < steps) step(s1, s0, st + 1);
        }
    } else {
        // (the workgroup's rows are the wavefront's: every tile of the walk touches them)
        for (int v = v0 + kw, st = 0; v < v1; v += KW, ++st) {  // wavefront-uniform
            const bool more = v + KW < v1, cut = !rw.inside(a, v, wfirst, wlast);
            pf_wait<0>();  // K and V are in
            if (cut && any_bad(sb1)) {
                mark_bad(sb1, v);
                pf_wait<0>();  // (its reads are done)
                drop_bad(sb1);
                pf_wait<0>();
            }
            // both into registers, so that the next ones have the whole step to arrive
            uint32_t kat[KS];
            h8 x[KS], vx[2 * DT];
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
                kat[ks] = (uint32_t)(uintptr_t)(lds_void *)(void *)(sb + ka[ks]);
#pragma unroll
            for (int k = 0; k < 2 * DT; ++k) vx[k] = v_operand(sb1, k / 2, k % 2);
            lds_read16(kat, x);
            pf_wait<0>();  // (read)
            if (more) {
                const Pages next = page;
                page = page_of(st + 2);
                asm volatile("" ::: "memory");
                copy(a.k, sb, st + 1, next, true);
                copy(a.v, sb1, st + 1, next, false);
            }
            f16v s = products(x);
            refer(s, v, cut);
            weights(s);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int s2 = 0; s2 < 2; ++s2) {
                    const h8 y = vx[2 * dt + s2];
                    o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(y, ph[s2], o[dt], 0, 0, 0);
                    o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(y, pl[s2], o[dt], 0, 0, 0);
                }
        }
    }
}

// The outputs of a workgroup's walks (or its chunk's states): 0, or NaN where one of this thread's is
// not finite.
template <int D, int RT, int KW, int AHEAD>
__device__ __forceinline__ float rows_put(const RowsArgs &a, const RowsParts &pt,
                                          const RowsShare &sh, int tid, uint8_t *sb, uint8_t *sb1,
                                          float (*mrg_m)[PF_T], float (*mrg_l)[PF_T], float c,
                                          float lsum, const f16v (&o)[D / 32]) {
    using F = RowsForm<D, RT, KW, AHEAD>;
    constexpr int NT = F::NT, DT = D / 32, OROW = F::OROW, MRG_W = F::MRG_W;
    const RowTile &rw = sh.rw;
    const bool whole = rw.ntiles <= pt.chunk_tiles;  // the results themselves, not a part
    const int g = sh.g, per = a.qheads / a.kvheads, tile_id = sh.tile, chunk = sh.chunk;
    const RowsWave me = RowsWave::of<RT>(a, sh, tid);
    const int rt = me.rt, t = me.t, hh = me.hh, wave = me.kw * RT + rt;
    const int myrow = me.row, myhead = me.head, prow = me.pos;
    float z = 0.0f;
    lsum += swap32_f(lsum);

    // lane (t, hh) holds O[row t][32 dt + 8 (r / 4) + 4 hh + r % 4] in o[dt][r]
    if constexpr (KW == 1) {
        // (never cut) each lane its row's halves of 8: 16-byte stores, the Q8_0 of a block
        // from the pair of lanes that holds it
        const int lr = 32 * rt + t;
        const float inv = 1.0f / lsum;
        const size_t off = ((size_t)myrow * a.qheads + myhead) * D;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            float y[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) y[r] = prow < 0 ? 0.0f : o[dt][r] * inv;
            uint32_t q[4];
            uint16_t dbits;
            int sum;
            if (a.qs) quant_block_pair16(y, q, dbits, sum);  // every lane
            if (lr >= rw.pairs) continue;
#pragma unroll
            for (int r = 0; r < 16; ++r) z = fmaf(y[r], 0.0f, z);
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4)
                *(f4 *)(a.attn + off + 32 * dt + 8 * r4 + 4 * hh) =
                    (f4){y[4 * r4], y[4 * r4 + 1], y[4 * r4 + 2], y[4 * r4 + 3]};
            if (!a.qs) continue;
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4)
                *(uint32_t *)(a.qs + off + 32 * dt + 8 * r4 + 4 * hh) = q[r4];
            if (hh == 0) {
                a.d[off / SI_QK + dt] = dbits;
                if (a.bsum) a.bsum[off / SI_QK + dt] = (int16_t)sum;
            }
        }
        return z;
    }
    pf_wait<0>();  // no copy in flight (a wavefront without tiles never waited for its own)
    __syncthreads();  // every wavefront is done with the stages
    const auto mo = [&](int w) {  // [row][OROW] of a wavefront
        return (float *)(w < MRG_W ? sb : sb1) + (w % MRG_W) * (PF_T * OROW);
    };
    if (hh == 0 && KW > 1) {
        mrg_m[wave][t] = c;
        mrg_l[wave][t] = lsum;
    }
    if (32 * rt + t < rw.pairs)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4)
                *(f4 *)(mo(wave) + t * OROW + 32 * dt + 8 * r4 + 4 * hh) =
                    (f4){o[dt][4 * r4], o[dt][4 * r4 + 1], o[dt][4 * r4 + 2], o[dt][4 * r4 + 3]};
    __syncthreads();
    // a row's factors for its KW states, in mrg_m: 2^(c_k - largest), over the sum where
    // the results come from this workgroup alone
    if (tid < rw.pairs && KW > 1) {
        const int w0 = tid >> 5, tr = tid & 31;
        float M = -INFINITY, l = 0.0f, f[KW];
#pragma unroll
        for (int k = 0; k < KW; ++k) M = fmaxf(M, mrg_m[k * RT + w0][tr]);
        const float ref = M == -INFINITY ? 0.0f : M;
#pragma unroll
        for (int k = 0; k < KW; ++k) {
            f[k] = __builtin_amdgcn_exp2f(mrg_m[k * RT + w0][tr] - ref);
            l = fmaf(mrg_l[k * RT + w0][tr], f[k], l);
        }
        if (!whole) {
            const size_t at = part_row(pt, a.kvheads, tile_id, g, chunk, tid);
            pt.m[2 * at] = M;
            pt.m[2 * at + 1] = l;
        }
        const float inv = whole ? 1.0f / l : 1.0f;
#pragma unroll
        for (int k = 0; k < KW; ++k) mrg_m[k * RT + w0][tr] = some(f[k] * inv);
    }
    __syncthreads();
    // 4 consecutive elements of a row per thread: merge the KW states, quantize (8 lanes
    // hold one Q8_0 block, qwen_one_layer.c:272)
    for (int e = tid; e < rw.pairs * (D / 4); e += NT) {
        const int lr = e / (D / 4), dd = 4 * (e % (D / 4)), w0 = lr >> 5, tr = lr & 31;
        float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < KW; ++k) {
            const int w = k * RT + w0;
            const f4 v = *(const f4 *)(mo(w) + tr * OROW + dd);
            const float f = mrg_m[KW > 1 ? w : 0][tr];
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = fmaf(v[i], f, y[i]);
        }
        if (!whole) {
            *(f4 *)(pt.o + part_row(pt, a.kvheads, tile_id, g, chunk, lr) * D + dd) =
                (f4){y[0], y[1], y[2], y[3]};
        } else {
            const int pair = rw.pair0 + lr;
            rows_store<D>(a, rw.row0 + pair / per, g * per + pair % per, dd, rw.p0 + pair / per, y);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) z = fmaf(y[i], 0.0f, z);
    }
    return z;
}

// The second walk and its outputs.
template <int D, int RT, int KW, int AHEAD, bool ONE, int PAGE>
__device__ __forceinline__ void rows_again(RowsArgs a, RowsParts pt, RowsShare sh, int tid,
                                                     uint8_t *sb, uint8_t *sb1,
                                                     float (*mrg_m)[PF_T], float (*mrg_l)[PF_T]) {
    float c, lsum;
    f16v o[D / 32];
    rows_walk<D, RT, KW, AHEAD, ONE, PAGE, true>(a, sh, tid, sb, sb1, nullptr, c, lsum, o);
    rows_put<D, RT, KW, AHEAD>(a, pt, sh, tid, sb, sb1, mrg_m, mrg_l, c, lsum, o);
}

template <int D, int RT, int KW, int AHEAD, bool ONE, int PAGE>
__global__ void __launch_bounds__(RT * KW * 64) __attribute__((amdgpu_waves_per_eu(2)))
k_attn_rows(RowsArgs a, RowsParts pt) {
    using F = RowsForm<D, RT, KW, AHEAD>;
    __shared__ __attribute__((aligned(16))) uint8_t sb[F::SB];
    __shared__ __attribute__((aligned(16))) uint8_t sb1[F::DB ? 16 : F::SB];
    __shared__ float mrg_m[KW > 1 ? F::NWV : 1][PF_T], mrg_l[KW > 1 ? F::NWV : 1][PF_T];
    __shared__ int bad_step[3];  // whether a cut step's V holds infinities or NaN (of two steps in
                                 // turn); whether outputs are not finite

    const int tid = threadIdx.x;
    if (tid == 0) bad_step[2] = 0;  // (a barrier of the walk or the outputs lies before its use)
    // KV groups side by side: one group's tiles on the same XCDs where their count
    // divides 8
    RowsShare sh;
    sh.g = blockIdx.x % a.kvheads;
    sh.tile = blockIdx.x / a.kvheads / pt.chunks;
    sh.chunk = blockIdx.x / a.kvheads % pt.chunks;
    if (!find_tile<ONE, F::NT>(a, 32 * RT, sh.tile, sh.rw)) return;
    sh.v0 = sh.chunk * pt.chunk_tiles, sh.v1 = min(sh.rw.ntiles, sh.v0 + pt.chunk_tiles);
    if (sh.chunk > 0 && sh.v0 >= sh.v1) return;

    float c, lsum;
    f16v o[D / 32];
    rows_walk<D, RT, KW, AHEAD, ONE, PAGE, false>(a, sh, tid, sb, sb1, bad_step, c, lsum, o);
    const float z =
        rows_put<D, RT, KW, AHEAD>(a, pt, sh, tid, sb, sb1, mrg_m, mrg_l, c, lsum, o);
    if (__ballot(!(z == 0.0f)) && (tid & 63) == 0) bad_step[2] = 1;
    __syncthreads();
    if (bad_step[2]) {
        // (a lane's numbers are made anew, not kept in registers through the first walk)
        int again = tid;
        asm volatile("" : "+v"(again));
        rows_again<D, RT, KW, AHEAD, ONE, PAGE>(a, pt, sh, again, sb, sb1, mrg_m, mrg_l);
    }
}

// ---------------------------------------------------------------------------
// The chunks' states of tiles that were cut: grid (tiles x KV groups, rows), 4 values of a
// row per thread, its chunks taken G ways (G > 1: they meet in LDS, in their order).
// Latency bounds it: out = sum_k 2^(m_k - m) o_k / sum_k 2^(m_k - m) l_k, a row's parts from
// the caches, four loads in flight; 3.0 us for 14 rows of 64 in 7 chunks, 4.6 us for
// 24 rows of 128 in 64 chunks (8 ways; one way 12).
// ---------------------------------------------------------------------------
constexpr int RM_T = 256;
template <int D, bool ONE, int G>
__global__ void __launch_bounds__(RM_T) k_attn_rows_merge(RowsArgs a, RowsParts pt,
                                                          int tile_rows) {
    constexpr int LANES = D / 4, ROWS = RM_T / (LANES * G);  // of a workgroup
    static_assert(ROWS >= 1, "a row's threads fit a workgroup");
    const int g = blockIdx.x % a.kvheads, tile_id = blockIdx.x / a.kvheads;
    RowTile rw;
    if (!find_tile<ONE, RM_T>(a, tile_rows, tile_id, rw) || rw.ntiles <= pt.chunk_tiles) return;
    const int grp = threadIdx.x / LANES, dd = 4 * (threadIdx.x % LANES);
    const int way = grp / ROWS, lr = blockIdx.y * ROWS + grp % ROWS;
    const bool mine = way < G && lr < rw.pairs;  // whole groups of 8 lanes
    const int n = (rw.ntiles + pt.chunk_tiles - 1) / pt.chunk_tiles;
    float M = -INFINITY, l = 0.0f, y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (mine) {
        constexpr int U = 4;  // chunks whose loads are in flight together
        for (int k0 = way; k0 < n; k0 += U * G) {
            float m[U], s[U];
            f4 v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {  // (past the last: it again, of no weight)
                const size_t at = part_row(pt, a.kvheads, tile_id, g, min(k0 + u * G, n - 1), lr);
                m[u] = k0 + u * G < n ? pt.m[2 * at] : -INFINITY;
                s[u] = pt.m[2 * at + 1];
                v[u] = *(const f4 *)(pt.o + at * D + dd);
            }
            float to = M;
#pragma unroll
            for (int u = 0; u < U; ++u) to = fmaxf(to, m[u]);
            const float ref = to == -INFINITY ? 0.0f : to;
            const float old = some(__builtin_amdgcn_exp2f(M - ref));
            M = to;
            l *= old;
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] *= old;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (k0 + u * G >= n) continue;
                // (of a chunk that the row sees nothing of all is 0; of one whose scores are NaN
                // the reference is as low, and the sum NaN)
                const float f = some(__builtin_amdgcn_exp2f(m[u] - ref));
                l = fmaf(s[u], f, l);
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = fmaf(v[u][i], f, y[i]);
            }
        }
    }
    if constexpr (G > 1) {
        __shared__ float all_m[G][ROWS], all_l[G][ROWS];
        __shared__ f4 all_y[G][ROWS * LANES];
        const int at = threadIdx.x % (ROWS * LANES);
        if (way < G) {
            if (dd == 0) {
                all_m[way][grp % ROWS] = M;
                all_l[way][grp % ROWS] = l;
            }
            all_y[way][at] = (f4){y[0], y[1], y[2], y[3]};
        }
        __syncthreads();
        if (way > 0 || !mine) return;
#pragma unroll
        for (int w = 0; w < G; ++w) M = fmaxf(M, all_m[w][grp % ROWS]);
        const float ref = M == -INFINITY ? 0.0f : M;
        l = y[0] = y[1] = y[2] = y[3] = 0.0f;
#pragma unroll
        for (int w = 0; w < G; ++w) {
            const float f = some(__builtin_amdgcn_exp2f(all_m[w][grp % ROWS] - ref));
            l = fmaf(all_l[w][grp % ROWS], f, l);
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = fmaf(all_y[w][at][i], f, y[i]);
        }
    }
    if (!mine) return;
    const float inv = 1.0f / l;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] *= inv;
    const int per = a.qheads / a.kvheads, pair = rw.pair0 + lr;
    rows_store<D>(a, rw.row0 + pair / per, g * per + pair % per, dd, rw.p0 + pair / per, y);
}

// ---------------------------------------------------------------------------
// How a call is cut
// ---------------------------------------------------------------------------
struct RowsPlan {
    bool one;    // a tile a sequence at most
    int rt, kw;  // wavefronts of a workgroup: 32-row tiles x K/V tiles
    int tiles;   // at most
    int chunks, chunk_tiles, rows;
    size_t parts() const { return chunks > 1 ? (size_t)tiles * chunks : 0; }
    long long items() const { return (long long)tiles * chunks; }
};

static RowsPlan rows_plan(const RowsArgs &a) {
    RowsPlan p;
    const int per = a.qheads / a.kvheads;
    const long long pairs = (long long)a.max_new * per;
    p.one = pairs <= 64;
    // Wavefronts of a workgroup.  Rows of a sequence that fill one or two 32-row tiles: a
    // workgroup for all of them, so that K and V are read once (16 sequences of 1-8 rows of 7
    // heads 32.0 us, a workgroup for each tile 35.3).  More (prompts): while the
    // 32-row tiles are few each is a workgroup's, its walk taken four ways; past that four
    // tiles share each staged K/V tile (us, 1x4 | 4x1: 28/4 heads of 128, 1000 rows 39 | 50,
    // 2048 (1792 tiles) 94 | 97, 3000 in a window of 1024 (2628) 127 | 107, 8000 of 2048
    // 500 | 422; 14/2 of 64, 2048 rows 31 | 67, 4000 in 1024 (1750) 49 | 58, 8000 of 2048
    // (3500) 144 | 148).
    const long long tiles32 = ((long long)a.max_rows * per + 31) / 32 * a.kvheads;
    p.rt = pairs <= 32 ? 1 : pairs <= 64 ? 2 : tiles32 < (a.hdim <= 64 ? 3500 : 1800) ? 1 : 4;
    p.kw = p.rt == 4 ? 1 : p.rt == 2 ? 2 : 4;
    const int rows = 32 * p.rt;
    // (of a batch of several sequences the tiles are about max_rows' and at most one more each)
    const int about =
        std::max(1, p.one ? a.nseq : (int)(((long long)a.max_rows * per + rows - 1) / rows));
    p.tiles = p.one ? a.nseq
                    : (int)((long long)a.max_rows * per / rows) + std::min(a.nseq, a.max_rows);
    p.rows = (int)std::min<long long>(rows, pairs);
    // K/V tiles that a tile's rows can see: the sinks', and a window's of every row
    const long long span = std::min<long long>(a.max_ctx, (long long)a.window + rows / per + 1);
    const int most = (int)std::min<long long>((a.max_ctx + PF_T - 1) / PF_T, span / PF_T + 2) +
                     (a.sinks + PF_T - 1) / PF_T;
    const long long base = (long long)a.kvheads * about;
    // Chunks so that there are 256 workgroups of one row tile (one a CU: two halve the walks
    // but double the states to merge; us, 256 | 512 | 1024 workgroups: 64 x 4096 of 28/4 heads
    // of 128 90 | 93 | 107, 2 x 65536 of 12/2 28.9 | 30.3 | 39.9, 100 rows after 1000 19.6 |
    // 21.0 | -), 512 of two, whose fewer wavefronts share a K/V tile (16 sequences of 1-8 rows
    // 34.8 | 32.3 | 41).  Workgroups of four tiles are more than that from the start.
    long long chunks = p.rt == 4 ? 1 : (p.rt == 1 ? 256 : 512) / base;
    // (a step of a workgroup at least, and as many states as there is room for)
    const size_t state = (size_t)p.tiles * a.kvheads * p.rows * (a.hdim + 2) *
                         sizeof(float);
    chunks = std::min<long long>(chunks, most / p.kw);
    if (state > 0) chunks = (long long)std::min<size_t>((size_t)std::max(chunks, 0LL),
                                                        a.ws_most / state);
    chunks = std::max(1LL, chunks);
    p.chunk_tiles = (int)((most + chunks - 1) / chunks);
    p.chunks = (most + p.chunk_tiles - 1) / p.chunk_tiles;
    return p;
}

size_t attn_rows_workspace(const RowsArgs &a) {
    const RowsPlan p = rows_plan(a);
    return p.parts() * a.kvheads * p.rows * (a.hdim + 2) * sizeof(float);
}

bool attn_rows_fits(const RowsArgs &a) {
    const RowsPlan p = rows_plan(a);
    // (a launch's threads are counted in 32 bits)
    return p.items() * a.kvheads * p.rt * p.kw * 64 < (1LL << 32);
}

void launch_attn_rows_paged(const RowsArgs &a, void *workspace, hipStream_t st) {
    const RowsPlan p = rows_plan(a);
    RowsParts pt = {};
    pt.chunks = p.chunks;
    pt.chunk_tiles = p.chunk_tiles;
    pt.rows = p.rows;
    pt.o = (float *)workspace;
    pt.m = pt.o + p.parts() * a.kvheads * p.rows * a.hdim;
    const dim3 grid((unsigned)(p.items() * a.kvheads)), block(p.rt * p.kw * 64);
#define CALL(DIM, RT, KW, AHEAD, ONE, PAGE) \
    SI_LAUNCH((k_attn_rows<DIM, RT, KW, AHEAD, ONE, PAGE>), grid, block, 0, st, a, pt)
#define PAGES(DIM, RT, KW, AHEAD, ONE)                                              \
    if (a.pg.shift >= 5) CALL(DIM, RT, KW, AHEAD, ONE, 32);                          \
    else if (a.pg.shift == 4 && DIM != 96) CALL(DIM, RT, KW, AHEAD, ONE, (DIM == 96 ? 1 : 16)); \
    else CALL(DIM, RT, KW, AHEAD, ONE, 1)
#define DIMS(DIM)                                              \
    if (p.rt == 1 && p.one) { PAGES(DIM, 1, 4, 1, true); }    \
    else if (p.rt == 1) { PAGES(DIM, 1, 4, 1, false); }       \
    else if (p.rt == 2) { PAGES(DIM, 2, 2, 1, true); }        \
    else { PAGES(DIM, 4, 1, 2, false); }
    // (a row's chunks 8 ways where there are many: 2 x 65536 positions in 64, 28.9 us against 36.7)
#define MERGE(DIM, ONE, G)                                                                    \
    SI_LAUNCH((k_attn_rows_merge<DIM, ONE, G>),                                                 \
              dim3((unsigned)(p.tiles * a.kvheads),                                             \
                   (p.rows - 1) / (RM_T / (DIM / 4 * G)) + 1),                                  \
              dim3(RM_T), 0, st, a, pt, 32 * p.rt)
#define MERGES(DIM)                                          \
    if (p.chunks > 8) {                                      \
        if (p.one) MERGE(DIM, true, 8);                      \
        else MERGE(DIM, false, 8);                           \
    } else if (p.chunks > 1) {                               \
        if (p.one) MERGE(DIM, true, 1);                      \
        else MERGE(DIM, false, 1);                           \
    }
    switch (a.hdim) {
        case 32: DIMS(32); MERGES(32); break;
        case 64: DIMS(64); MERGES(64); break;
        case 96: DIMS(96); MERGES(96); break;
        default: DIMS(128); MERGES(128); break;
    }
#undef MERGES
#undef MERGE
#undef DIMS
#undef PAGES
#undef CALL
}

}  // namespace si
