// si_tiles.hpp -- what the attention kernels over 32 x 32 tiles share: a K and a V tile in
// LDS, the split of 32-bit values into fp16 halves, the waits of copies into LDS.
#pragma once
#include "si_device.hpp"

namespace si {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef _Float16 pf_h2 __attribute__((ext_vector_type(2)));
typedef float pf_f2 __attribute__((ext_vector_type(2)));

constexpr int PF_T = 32;      // query rows per wavefront, positions per K/V tile
constexpr int PF_OPAD = 4;    // floats of padding per merged output row

// LDS slot (16-byte unit within the row) of chunk c of tile row r: the 16
// rows a score operand read takes together, and the 4 rows x 4 chunks of a
// transposing read, spread over the 64 banks
template <int D>
__device__ __forceinline__ int pf_k_slot(int r, int c) {
    if (D == 128) return c ^ (r & 15);
    if (D == 64) return c ^ ((r >> 1) & 7);
    if (D == 32) return c ^ ((r >> 2) & 3);
    const int s = c + ((r >> 2) & 3);  // 12 chunks: a rotation
    return s >= D / 8 ? s - D / 8 : s;
}
template <int D>
__device__ __forceinline__ int pf_v_slot(int r, int c) {
    if (D == 128) return c ^ ((r & 3) << 2);
    if (D == 64) return c ^ (((r >> 1) & 1) << 2);
    return c;  // 4 rows already cover the banks
}
// the chunk whose slot is s
template <int D>
__device__ __forceinline__ int pf_k_chunk(int r, int s) {
    if (D != 96) return pf_k_slot<D>(r, s);  // an XOR
    const int c = s - ((r >> 2) & 3);
    return c < 0 ? c + D / 8 : c;
}

// (fmaxf of matrix results would first canonicalise each; a must come from an
// ordinary operation on those results)
__device__ __forceinline__ float max3_f(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
// two values as fp16 hi + lo halves (hi rounded to nearest, lo = x - hi by a
// mixed-precision fma; the plain conversion to hi reads both values first)
__device__ __forceinline__ void split_pair(float x0, float x1, pf_h2 &hi, pf_h2 &lo) {
    hi = __builtin_convertvector((pf_f2){x0, x1}, pf_h2);
    float l0, l1;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(l0) : "v"(hi), "v"(x0));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
        : "=v"(l1)
        : "v"(hi), "v"(x1));
    lo = __builtin_convertvector((pf_f2){l0, l1}, pf_h2);
}

// at most VM vector-memory operations of this wavefront outstanding, its LDS
// reads complete
template <int VM>
__device__ __forceinline__ void pf_wait() {
    static_assert(VM <= 63, "vmcnt holds 6 bits");
    __builtin_amdgcn_s_waitcnt((VM & 15) | ((VM >> 4) << 14) | (7 << 4));
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void pf_barrier() {
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// N 16-byte reads of LDS at the given addresses, complete on return.  As inline assembly,
// which the compiler does not know to read LDS: before its own reads it would wait for
// every copy into LDS under way, also those that go elsewhere.  The caller has waited for
// the bytes themselves.
template <int N>
__device__ __forceinline__ void lds_read16(const uint32_t (&at)[N], h8 (&x)[N]) {
    static_assert(N == 2 || N == 4 || N == 6 || N == 8, "the head dims' k-steps");
    if constexpr (N == 2)
        asm volatile("ds_read_b128 %0, %2\n\tds_read_b128 %1, %3\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(x[0]), "=&v"(x[1])
                     : "v"(at[0]), "v"(at[1])
                     : "memory");
    if constexpr (N == 4)
        asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %5\n\t"
                     "ds_read_b128 %2, %6\n\tds_read_b128 %3, %7\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3])
                     : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3])
                     : "memory");
    if constexpr (N == 6)
        asm volatile("ds_read_b128 %0, %6\n\tds_read_b128 %1, %7\n\t"
                     "ds_read_b128 %2, %8\n\tds_read_b128 %3, %9\n\t"
                     "ds_read_b128 %4, %10\n\tds_read_b128 %5, %11\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(x[4]),
                       "=&v"(x[5])
                     : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "v"(at[4]), "v"(at[5])
                     : "memory");
    if constexpr (N == 8)
        asm volatile("ds_read_b128 %0, %8\n\tds_read_b128 %1, %9\n\t"
                     "ds_read_b128 %2, %10\n\tds_read_b128 %3, %11\n\t"
                     "ds_read_b128 %4, %12\n\tds_read_b128 %5, %13\n\t"
                     "ds_read_b128 %6, %14\n\tds_read_b128 %7, %15\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(x[4]),
                       "=&v"(x[5]), "=&v"(x[6]), "=&v"(x[7])
                     : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "v"(at[4]), "v"(at[5]),
                       "v"(at[6]), "v"(at[7])
                     : "memory");
}
// lds_copy16 at soff more, wavefront-uniform; AUX: its cache policy
template <int AUX>
__device__ __forceinline__ void lds_copy16(__amdgpu_buffer_rsrc_t r, uint8_t *lds, uint32_t voff,
                                           int soff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void *)lds, 16, voff, soff, 0, AUX);
}
// lds_copy16 from an address of its own for each lane
typedef __attribute__((address_space(1))) void global_void;
__device__ __forceinline__ void lds_copy16_at(const uint8_t *p, uint8_t *lds) {
    __builtin_amdgcn_global_load_lds((global_void *)p, (lds_void *)lds, 16, 0, 0);
}

}  // namespace si
