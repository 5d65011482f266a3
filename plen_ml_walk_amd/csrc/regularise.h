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
template <int DT> struct Chunk { typename Elem<DT>::T v[8]; };
template <int DT> static __device__ __forceinline__ Chunk<DT> load_whole(const typename Elem<DT>::T *p) {
    Chunk<DT> c;
    __builtin_memcpy(&c, p, sizeof c);
    return c;
}
// the first `valid` elements (the rest: zeros).  A part of a chunk goes as four, two and one elements.
template <int DT> static __device__ __forceinline__ Chunk<DT> load_chunk(const typename Elem<DT>::T *p, int valid) {
    typedef typename Elem<DT>::T T;
    if (valid >= 8) return load_whole<DT>(p);
    T four[4] = {}, two[2] = {}, one = (T)0.f;
    if (valid & 4) __builtin_memcpy(four, p, sizeof four);
    if (valid & 2) __builtin_memcpy(two, p + (valid & 4), sizeof two);
    if (valid & 1) one = p[valid & 6];
    const T rest[4] = {valid & 2 ? two[0] : one, two[1], valid & 2 ? one : (T)0.f, (T)0.f};
    Chunk<DT> c;
#pragma unroll
    for (int e = 0; e < 4; e++) { c.v[e] = valid & 4 ? four[e] : rest[e]; c.v[4 + e] = valid & 4 ? rest[e] : (T)0.f; }
    return c;
}
template <int DT> static __device__ __forceinline__ void store_whole(typename Elem<DT>::T *p, const float (&v)[8]) {
    Chunk<DT> c;
#pragma unroll
    for (int e = 0; e < 8; e++) c.v[e] = (typename Elem<DT>::T)v[e];
    __builtin_memcpy(p, &c, sizeof c);
}
template <int DT> static __device__ __forceinline__ void store_chunk(typename Elem<DT>::T *p, int valid, const float (&v)[8]) {
    typedef typename Elem<DT>::T T;
    if (valid >= 8) { store_whole<DT>(p, v); return; }
    T c[8], rest[3];
#pragma unroll
    for (int e = 0; e < 8; e++) c[e] = (T)v[e];
    if (valid & 4) __builtin_memcpy(p, c, 4 * sizeof(T));
#pragma unroll
    for (int e = 0; e < 3; e++) rest[e] = valid & 4 ? c[4 + e] : c[e];
    if (valid & 2) __builtin_memcpy(p + (valid & 4), rest, 2 * sizeof(T));
    if (valid & 1) p[valid & 6] = valid & 2 ? rest[2] : rest[0];
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
// ... of the 8 elements from element i on
static __device__ __forceinline__ uint32_t chunk_mask(const Draw &d, int64_t i) {
    const uint32_t block = (uint32_t)(i >> 3), shift = (uint32_t)i & 7u;
    uint32_t m = block_mask(d, block);
    if (shift) m = (m | block_mask(d, block + 1) << 8) >> shift;
    return m;
}
static __device__ __forceinline__ bool kept(const Draw &d, int64_t i) { return block_mask(d, (uint32_t)(i >> 3)) >> (i & 7) & 1u; }

// ---- group norm: arguments and plans as the host hands them to the kernels (quotients and scales worked out once)
struct NormArgs {
    const void *x, *dy, *w, *b;
    void *out;
    double2 *stats;                  // [N][G]: mean m of the masked, unscaled input and r = scale / sqrt(scale^2 variance + eps): the normalised value is (x - m) r, also with dropout
    const uint64_t *rng;
    uint64_t *used;
    int64_t N, x_stride, dy_stride, size;          // size = L C
    double inv_count, scale, eps;                  // 1 / (L D); dropout's factor
    int C, G, D, act, site;
    uint32_t cut;
    float inv_D, inv_C;
};
// i / n for 0 <= i < 2^20, with 1 / n in float: (i + 1/2) / n is at least 1 / (2 n) away from the next integer, the product's error is less than i 2^-22 / n
static __device__ __forceinline__ int small_quotient(int i, float inv_n) { return (int)(((float)i + 0.5f) * inv_n); }

// rows of one position: 2^team_log lanes per (row, group); a workgroup covers gb neighbouring groups of rb rows per turn
struct RowPlan { int team_log, gb, rb, trips; float inv_gb; };
struct RowLaunch { RowPlan P; int K, NT; dim3 grid; };
// many positions.  A slab as `rows` rows of `ncol` chunk columns (q positions to a row); bcol columns in a workgroup, R rows per turn of it
struct MapPlan { int q, ncol, bcol, col_blocks, R, splits; int64_t rows, rows_per; int lanes_log, row_blocks; int64_t apply_rows; float inv_bcol; };
struct MapLaunch { MapPlan P; dim3 sums; int NT; unsigned stat_blocks, apply_blocks; size_t lds; };

// one per pair of element types (x and results, parameters), in regularise_norm.hip
struct NormEntry {
    void (*row_forward)(const NormArgs &, const RowLaunch &, hipStream_t);
    void (*row_backward)(const NormArgs &, const RowLaunch &, float *part, hipStream_t);
    void (*map_forward)(const NormArgs &, const MapLaunch &, double2 *part, hipStream_t);
    void (*map_backward)(const NormArgs &, const MapLaunch &, double2 *part, float2 *means, float *params, void *dw, void *db, hipStream_t);
    void (*params)(const NormArgs &, const float *part, int rows, void *dw, void *db, hipStream_t);
};
const NormEntry &plenreg_norm_f32_f32();
const NormEntry &plenreg_norm_bf16_f32();
const NormEntry &plenreg_norm_bf16_bf16();
const NormEntry &plenreg_norm_f16_f32();
const NormEntry &plenreg_norm_f16_f16();

#endif
