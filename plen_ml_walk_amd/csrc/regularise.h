// regularise.h -- what regularise.hip (C ABI, launch plans, dropout) and regularise_norm.hip (group norm, compiled once per pair of element types) share.
#ifndef PLEN_REGULARISE_H
#define PLEN_REGULARISE_H
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "../../include/plenreg.h"
#ifdef __HIP_DEVICE_COMPILE__
#define PHILOX_XOR3(a, b, c) __builtin_amdgcn_bitop3_b32((a), (b), (c), 0x96)          // one instruction instead of two
#endif
#include "philox.h"

// ---- element types: arithmetic is in 32 bits, each result is rounded once, when it is stored
template <int DT> struct Elem;
template <> struct Elem<PLENREG_F32> { typedef float T; };
template <> struct Elem<PLENREG_BF16> { typedef __bf16 T; };
template <> struct Elem<PLENREG_F16> { typedef _Float16 T; };

// ---- 8 neighbouring elements, the unit of every kernel: 16 bytes of a 16-bit type, 32 of float32; aligned like one element only (rows of odd
//      widths begin anywhere; the wide loads take any address)
//      (Held as 32-bit words: 16-bit elements would be taken apart, and waited for, at the end of every block that a load is carried out of.)
template <int DT> struct Chunk {
    uint32_t w[DT == PLENREG_F32 ? 8 : 4];
    __device__ __forceinline__ float get(int e) const {          // (e is a constant where this is inlined)
        if constexpr (DT == PLENREG_F32) return __uint_as_float(w[e]);
        else if constexpr (DT == PLENREG_BF16) return __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
        else return (float)__builtin_bit_cast(_Float16, (uint16_t)(e & 1 ? w[e >> 1] >> 16 : w[e >> 1]));
    }
};
template <int DT> static __device__ __forceinline__ Chunk<DT> pack(const float (&v)[8]) {
    typedef typename Elem<DT>::T Two __attribute__((ext_vector_type(2)));
    Chunk<DT> c;
    if constexpr (DT == PLENREG_F32) {
#pragma unroll
        for (int e = 0; e < 8; e++) c.w[e] = __float_as_uint(v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) c.w[e] = __builtin_bit_cast(uint32_t, Two{(typename Elem<DT>::T)v[2 * e], (typename Elem<DT>::T)v[2 * e + 1]});
    }
    return c;
}
template <int DT> static __device__ __forceinline__ Chunk<DT> load_whole(const typename Elem<DT>::T *p) {
    Chunk<DT> c;
    __builtin_memcpy(&c, p, sizeof c);
    return c;
}
template <int DT> static __device__ __forceinline__ void store_whole(typename Elem<DT>::T *p, const float (&v)[8]) {
    const Chunk<DT> c = pack<DT>(v);
    __builtin_memcpy(p, &c, sizeof c);
}
// the same past the caches (non-temporal): for tensors beyond what these hold, where keeping this one throws out others
typedef uint32_t Word4 __attribute__((ext_vector_type(4), aligned(2)));
template <int DT> static __device__ __forceinline__ Chunk<DT> stream_whole(const typename Elem<DT>::T *p) {
    Chunk<DT> c;
#pragma unroll
    for (int i = 0; i < (int)(sizeof c / 16); i++) {
        const Word4 t = __builtin_nontemporal_load((const Word4 *)p + i);
        c.w[4 * i] = t.x; c.w[4 * i + 1] = t.y; c.w[4 * i + 2] = t.z; c.w[4 * i + 3] = t.w;
    }
    return c;
}
template <int DT> static __device__ __forceinline__ void stream_store_whole(typename Elem<DT>::T *p, const float (&v)[8]) {
    const Chunk<DT> c = pack<DT>(v);
#pragma unroll
    for (int i = 0; i < (int)(sizeof c / 16); i++) __builtin_nontemporal_store(Word4{c.w[4 * i], c.w[4 * i + 1], c.w[4 * i + 2], c.w[4 * i + 3]}, (Word4 *)p + i);
}
// Part of a chunk goes as four, two and one elements.  Quad: four elements in one register value (an array here would be put into memory).
template <int SIZE> struct Quad;
template <> struct Quad<2> {
    typedef uint64_t Four; typedef uint32_t Two; typedef uint16_t One;
    static __device__ __forceinline__ Four join(Two two, One one, bool has_two) { return has_two ? (Four)two | (Four)one << 32 : (Four)one; }
    static __device__ __forceinline__ Two first(Four q) { return (Two)q; }
    static __device__ __forceinline__ One single(Four q, bool after_two) { return (One)(after_two ? q >> 32 : q); }
};
template <> struct Quad<4> {
    typedef uint32_t Four __attribute__((ext_vector_type(4)));
    typedef uint32_t Two __attribute__((ext_vector_type(2)));
    typedef uint32_t One;
    static __device__ __forceinline__ Four join(Two two, One one, bool has_two) { return has_two ? Four{two.x, two.y, one, 0u} : Four{one, 0u, 0u, 0u}; }
    static __device__ __forceinline__ Two first(Four q) { return q.xy; }
    static __device__ __forceinline__ One single(Four q, bool after_two) { return after_two ? q.z : q.x; }
};
// the first `valid` elements (the rest: zeros)
template <int DT> static __device__ __forceinline__ Chunk<DT> load_chunk(const typename Elem<DT>::T *p, int valid) {
    typedef Quad<sizeof(typename Elem<DT>::T)> Q;
    if (valid >= 8) return load_whole<DT>(p);
    typename Q::Four four = {};
    typename Q::Two two = {};
    typename Q::One one = 0;
    if (valid & 4) __builtin_memcpy(&four, p, sizeof four);
    if (valid & 2) __builtin_memcpy(&two, p + (valid & 4), sizeof two);
    if (valid & 1) __builtin_memcpy(&one, p + (valid & 6), sizeof one);
    const typename Q::Four rest = Q::join(two, one, valid & 2);
    struct { typename Q::Four lo, hi; } both = {valid & 4 ? four : rest, valid & 4 ? rest : (typename Q::Four){}};
    Chunk<DT> c;
    __builtin_memcpy(&c, &both, sizeof c);
    return c;
}
template <int DT> static __device__ __forceinline__ void store_chunk(typename Elem<DT>::T *p, int valid, const float (&v)[8]) {
    typedef typename Elem<DT>::T T;
    typedef Quad<sizeof(T)> Q;
    if (valid >= 8) { store_whole<DT>(p, v); return; }
    const Chunk<DT> c = pack<DT>(v);
    struct { typename Q::Four lo, hi; } both;
    __builtin_memcpy(&both, &c, sizeof c);
    if (valid & 4) __builtin_memcpy(p, &both.lo, sizeof both.lo);
    const typename Q::Four rest = valid & 4 ? both.hi : both.lo;
    const typename Q::Two two = Q::first(rest);
    const typename Q::One one = Q::single(rest, valid & 2);
    if (valid & 2) __builtin_memcpy(p + (valid & 4), &two, sizeof two);
    if (valid & 1) __builtin_memcpy(p + (valid & 6), &one, sizeof one);
}

// ---- the mask (plenreg.h): 16 bits of the stream per element, so one generator call serves a chunk.  Ten rounds of two 32 x 32 -> 64-bit products
//      per 8 elements stay below the memory time of 8 16-bit elements; 32 bits per element would not.
struct Draw { uint32_t call_lo, call_hi, tag, key_lo, key_hi, cut; };
static __device__ __forceinline__ Draw make_draw(const uint64_t *rng, int site, uint32_t cut) {
    const uint64_t seed = rng[0], call = rng[1];
    return Draw{(uint32_t)call, (uint32_t)(call >> 32), 16u + (uint32_t)site, (uint32_t)seed, (uint32_t)(seed >> 32), cut};
}
static __device__ __forceinline__ u4 block_words(const Draw &d, uint32_t block) { return philox4x32(block, d.call_lo, d.call_hi, d.tag, d.key_lo, d.key_hi); }
// bit e: is element e of the block of 8 elements kept?
static __device__ __forceinline__ uint32_t block_mask(const Draw &d, uint32_t block) {
    const u4 w = block_words(d, block);
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) m |= ((words[k] & 0xffffu) >= d.cut ? 1u << (2 * k) : 0u) | ((words[k] >> 16) >= d.cut ? 2u << (2 * k) : 0u);
    return m;
}
// the mask of the 8 elements from element i on.  M = 2: i is a multiple of 8, the block's words are kept and compared where the mask is used (two instructions an element);
// M = 1: any i, one bit per element; M = 0: nothing is dropped
template <int M> struct Mask;
template <> struct Mask<2> {
    u4 w;
    uint32_t cut;
    Mask() = default;
    __device__ __forceinline__ Mask(const Draw &d, int64_t i) : w(block_words(d, (uint32_t)(i >> 3))), cut(d.cut) {}
    __device__ __forceinline__ float keep(int e, float v) const {          // (e is a constant where this is inlined)
        const uint32_t word = e < 2 ? w.x : e < 4 ? w.y : e < 6 ? w.z : w.w;
        return (e & 1 ? word >> 16 : word & 0xffffu) >= cut ? v : 0.f;
    }
    __device__ __forceinline__ uint32_t bits() const {
        uint32_t m = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) m |= keep(e, 1.f) != 0.f ? 1u << e : 0u;
        return m;
    }
};
template <> struct Mask<1> {
    uint32_t m;
    Mask() = default;
    __device__ __forceinline__ Mask(const Draw &d, int64_t i) {
        const uint32_t block = (uint32_t)(i >> 3), shift = (uint32_t)i & 7u;
        m = block_mask(d, block);
        if (shift) m = (m | block_mask(d, block + 1) << 8) >> shift;
    }
    __device__ __forceinline__ float keep(int e, float v) const { return m >> e & 1u ? v : 0.f; }
    __device__ __forceinline__ uint32_t bits() const { return m; }
};
template <> struct Mask<0> {
    Mask() = default;
    __device__ __forceinline__ Mask(const Draw &, int64_t) {}
    __device__ __forceinline__ float keep(int, float v) const { return v; }
    __device__ __forceinline__ uint32_t bits() const { return 255u; }
};
static __device__ __forceinline__ bool kept(const Draw &d, int64_t i) { return block_mask(d, (uint32_t)(i >> 3)) >> (i & 7) & 1u; }

// ---- group norm: arguments and plans as the host hands them to the kernels (quotients and scales worked out once)
struct NormArgs {
    const void *x, *dy, *w, *b;
    void *out;
    double2 *stats;                  // [N][G]: mean m of the masked, unscaled input and r = scale / sqrt(scale^2 variance + eps): the normalised value is (x - m) r, also with dropout
    const uint64_t *rng;
    uint64_t *used;
    int64_t N, x_stride, dy_stride, size;          // size = L C
    double count, inv_count, scale, eps;           // L D and 1 / (L D); dropout's factor
    int C, G, D, act, site;
    uint32_t cut;
    float inv_D, inv_C;
};
// i / n for 0 <= i < 2^20, with 1 / n in float: (i + 1/2) / n is at least 1 / (2 n) away from the next integer, the product's error is less than i 2^-22 / n
static __device__ __forceinline__ int small_quotient(int i, float inv_n) { return (int)(((float)i + 0.5f) * inv_n); }

// rows of one position: 2^team_log lanes per (row, group); a workgroup covers gb neighbouring groups of rb rows per turn
struct RowPlan { int team_log, gb, rb, trips; float inv_gb; };
struct RowLaunch { RowPlan P; int K, NT; dim3 grid; bool stream; };
// rows too wide for that: grid of (n, group) pairs, and of the parameter gradients
#define WIDE_LOG 9
#define WIDE_NT (1 << WIDE_LOG)
struct WideLaunch { unsigned grid; dim3 params; bool stream; };
// many positions.  A slab as `rows` rows of `ncol` chunk columns (2^q_log positions to a row); bcol columns in a workgroup, R rows per turn of it; rows_per rows in a
// workgroup of the sums, apply_rows in one of the result; 2^lanes_log lanes join one group
struct MapPlan { int q_log, ncol, bcol, col_blocks, R, splits, lanes_log, chan_log, join_log, param_z; int64_t rows, rows_per, apply_rows; float inv_bcol; };
// slab: one workgroup does a slab by itself (the grid is `sums`, slabs along y)
// walks: a workgroup of the sums goes over more than one slab; lean: more than two workgroups of them to a compute unit (span_sums)
struct MapLaunch { MapPlan P; dim3 sums, apply; int NT, param_rows; unsigned stat_blocks; bool stream, slab, joins, walks, lean; };

// one per pair of element types (x and results, parameters), in regularise_norm.hip
struct NormEntry {
    void (*row_forward)(const NormArgs &, const RowLaunch &, hipStream_t);
    void (*row_backward)(const NormArgs &, const RowLaunch &, float *part, hipStream_t);
    void (*wide_forward)(const NormArgs &, const WideLaunch &, hipStream_t);
    void (*wide_backward)(const NormArgs &, const WideLaunch &, float *part, hipStream_t);
    void (*map_forward)(const NormArgs &, const MapLaunch &, double2 *part, hipStream_t);
    void (*map_backward)(const NormArgs &, const MapLaunch &, double2 *part, double2 *means, float *params, double *running, void *dw, void *db, hipStream_t);
    void (*params)(const NormArgs &, const float *part, int rows, void *dw, void *db, hipStream_t);
};
const NormEntry &plenreg_norm_f32_f32();
const NormEntry &plenreg_norm_bf16_f32();
const NormEntry &plenreg_norm_bf16_bf16();
const NormEntry &plenreg_norm_f16_f32();
const NormEntry &plenreg_norm_f16_f16();

#endif
