// si_rows.hip -- GQA attention of a ragged step's rows over a paged fp16 cache, with a
// sliding window and a few first positions that stay visible (attention_flash,
// attention_kernels.h:80-164, has one query and sees everything).
//
// A row at position p of its sequence sees position t <= p where t > p - window or
// t < sinks.
#include "si_device.hpp"
#include "si_kernels.hpp"

namespace si {

// A wavefront for each (row, head): lane l scores position l of each group of 64 visible
// ones, then the group's weights meet V, a lane holding two or one of the head's values.
__global__ void __launch_bounds__(64) k_attn_rows_plain(RowsArgs a) {
    __shared__ float w_lds[64];
    __shared__ size_t at_lds[64];
    const int r = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, D = a.hdim;
    int lo = 0, hi = a.nseq;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.start[mid] <= r) lo = mid;
        else hi = mid;
    }
    const int first = a.start[lo], n = a.start[lo + 1] - first;
    if (r < first || r - first >= min(n, a.max_new)) return;
    const int p = min(a.ctx[lo], a.max_ctx) - n + r - first;
    const int w0 = max(p - a.window + 1, 0), ns = min(a.sinks, w0);
    const int seen = p < 0 ? 0 : ns + p + 1 - w0;
    const float *q = a.q + ((size_t)r * a.qheads + h) * D;
    const int g = h / (a.qheads / a.kvheads), kvd = a.kvheads * D;
    float m = -INFINITY, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int j0 = 0; j0 < seen; j0 += 64) {
        const int j = min(j0 + lane, seen - 1), t = j < ns ? j : w0 + j - ns;
        const size_t at = a.pg.at<true>(lo, t, 0, kvd) + (size_t)g * D;
        float s = 0.0f;
        for (int d = 0; d < D; ++d) s = fmaf(q[d], h2f(a.k[at + d]), s);
        s = j0 + lane < seen ? s * a.scale2 : -INFINITY;
        float mx = m;
        for (int k = 0; k < 64; ++k) mx = fmaxf(mx, __shfl(s, k, 64));
        const float ref = mx == -INFINITY ? 0.0f : mx;
        const float w = exp2f(s - ref), alpha = exp2f(m - ref);
        m = mx;
        float sum = 0.0f;
        for (int k = 0; k < 64; ++k) sum += __shfl(w, k, 64);
        l = l * alpha + sum;
        o0 *= alpha;
        o1 *= alpha;
        __syncthreads();
        w_lds[lane] = w;
        at_lds[lane] = at;
        __syncthreads();
        for (int k = 0; k < min(64, seen - j0); ++k) {
            if (lane < D) o0 = fmaf(w_lds[k], h2f(a.v[at_lds[k] + lane]), o0);
            if (lane + 64 < D) o1 = fmaf(w_lds[k], h2f(a.v[at_lds[k] + lane + 64]), o1);
        }
    }
    const size_t off = ((size_t)r * a.qheads + h) * D;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int d = lane + 64 * e;
        const float y = d < D && seen ? (e ? o1 : o0) / l : 0.0f;
        uint16_t dbits;
        int sum;
        const int qv = quant_block_lane(y, dbits, sum);  // every lane
        if (d >= D) continue;
        a.attn[off + d] = y;
        if (!a.qs) continue;
        a.qs[off + d] = (int8_t)qv;
        if ((d & 31) == 0) {
            a.d[(off + d) / SI_QK] = dbits;
            if (a.bsum) a.bsum[(off + d) / SI_QK] = (int16_t)sum;
        }
    }
}

size_t attn_rows_workspace(const RowsArgs &a) {
    (void)a;
    return 0;
}

void launch_attn_rows_paged(const RowsArgs &a, void *workspace, hipStream_t st) {
    (void)workspace;
    SI_LAUNCH(k_attn_rows_plain, dim3(a.max_rows, a.qheads), dim3(64), 0, st, a);
}

}  // namespace si
