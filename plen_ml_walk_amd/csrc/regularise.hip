// regularise.hip -- dropout from the counter-based generator, group norm with an activation over channels-last data, and the two in one pass,
// with their gradients (gfx950).  C ABI: include/plenreg.h.  All three are bound by memory traffic at size and by launch latency when small.
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

static __device__ __forceinline__ float load_param(const void *p, int dtype, int i, float otherwise) {
    if (!p) return otherwise;
    return dtype == PLENREG_F32 ? ((const float *)p)[i] : dtype == PLENREG_BF16 ? (float)((const __bf16 *)p)[i] : (float)((const _Float16 *)p)[i];
}
static __device__ __forceinline__ void store_param(void *p, int dtype, int i, float v) {
    if (dtype == PLENREG_F32) ((float *)p)[i] = v;
    else if (dtype == PLENREG_BF16) ((__bf16 *)p)[i] = (__bf16)v;
    else ((_Float16 *)p)[i] = (_Float16)v;
}

// ---- 8 neighbouring elements, the unit of every kernel: 16 bytes of a 16-bit type, 32 of float32; aligned like one element only (rows of odd
//      widths begin anywhere; the wide loads take any address)
template <int DT> struct Chunk { typename Elem<DT>::T v[8]; };
template <int DT> static __device__ __forceinline__ Chunk<DT> load_chunk(const typename Elem<DT>::T *p, int valid) {
    Chunk<DT> c;
    if (valid >= 8) __builtin_memcpy(&c, p, sizeof c);
    else {
#pragma unroll
        for (int e = 0; e < 8; e++) c.v[e] = e < valid ? p[e] : (typename Elem<DT>::T)0.f;
    }
    return c;
}
template <int DT> static __device__ __forceinline__ void store_chunk(typename Elem<DT>::T *p, int valid, const float (&v)[8]) {
    Chunk<DT> c;
#pragma unroll
    for (int e = 0; e < 8; e++) c.v[e] = (typename Elem<DT>::T)v[e];
    if (valid >= 8) __builtin_memcpy(p, &c, sizeof c);
    else {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (e < valid) p[e] = c.v[e];
    }
}

// ---- the mask (plenreg.h): 16 bits of the stream per element, so one generator call serves a chunk.  Ten rounds of two 32 x 32 -> 64-bit products
//      per 8 elements stay below the memory time of 8 16-bit elements; 32 bits per element would not.
struct Draw { uint32_t call_lo, call_hi, tag, key_lo, key_hi, cut; float scale; };
static __device__ __forceinline__ Draw make_draw(const uint64_t *rng, int site, uint32_t cut) {
    const uint64_t seed = rng[0], call = rng[1];
    return Draw{(uint32_t)call, (uint32_t)(call >> 32), 16u + (uint32_t)site, (uint32_t)seed, (uint32_t)(seed >> 32), cut,
                cut < 65536u ? (float)(65536.0 / (65536.0 - (double)cut)) : 0.f};
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
// v[e] = kept ? v[e] scale : 0 for a whole block of 8 elements
static __device__ __forceinline__ void drop_block(const Draw &d, uint32_t block, float (&v)[8]) {
    const u4 w = block_words(d, block);
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float s = v[e] * d.scale;
        v[e] = ((e & 1 ? words[e >> 1] >> 16 : words[e >> 1] & 0xffffu) >= d.cut) ? s : 0.f;
    }
}
// ... of the 8 elements from element i on; aligned: i is known to be a multiple of 8
static __device__ __forceinline__ uint32_t chunk_mask(const Draw &d, int64_t i, bool aligned) {
    const uint32_t block = (uint32_t)(i >> 3), shift = (uint32_t)i & 7u;
    if (aligned || shift == 0) return block_mask(d, block);
    return (block_mask(d, block) | block_mask(d, block + 1) << 8) >> shift;
}
static __device__ __forceinline__ bool kept(const Draw &d, int64_t i) { return block_mask(d, (uint32_t)(i >> 3)) >> (i & 7) & 1u; }

// ---- dropout.  U chunks per thread: all loads are issued before the first mask is drawn.  In rows that are not contiguous (ROWS) a chunk that crosses
//      the end of a row is loaded element by element.
template <int DT, int U, bool ROWS> __global__ __launch_bounds__(256) void k_dropout(PlenRegDropout A) {
    typedef typename Elem<DT>::T T;
    const T *x = (const T *)A.x;
    T *y = (T *)A.y;
    const Draw d = make_draw(A.rng, A.site, A.cut);
    if (A.used && blockIdx.x == 0 && threadIdx.x == 0) { A.used[0] = A.rng[0]; A.used[1] = A.rng[1]; }
    const int64_t n = A.rows * A.cols, first = (int64_t)blockIdx.x * (256 * U);
    if (!ROWS && (first + 256 * U) * 8 <= n) {                     // every chunk of the workgroup is whole
        Chunk<DT> c[U];
#pragma unroll
        for (int u = 0; u < U; u++) c[u] = load_chunk<DT>(x + (first + u * 256 + threadIdx.x) * 8, 8);
#pragma unroll
        for (int u = 0; u < U; u++) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = (float)c[u].v[e];
            drop_block(d, (uint32_t)(first + u * 256 + threadIdx.x), v);
            store_chunk<DT>(y + (first + u * 256 + threadIdx.x) * 8, 8, v);
        }
        return;
    }
    for (int u = 0; u < U; u++) {
        const int64_t j = first + u * 256 + threadIdx.x, i = j << 3;
        if (i >= n) return;
        const int valid = n - i < 8 ? (int)(n - i) : 8;
        Chunk<DT> c;
        if (ROWS) {
            int64_t row = n >> 32 ? i / A.cols : (int64_t)((uint32_t)i / (uint32_t)A.cols), col = i - row * A.cols;
            if (col + valid <= A.cols) c = load_chunk<DT>(x + row * A.x_stride + col, valid);
            else
                for (int e = 0; e < 8; e++) {
                    c.v[e] = e < valid ? x[row * A.x_stride + col] : (T)0.f;
                    if (++col == A.cols) { col = 0; row++; }
                }
        } else c = load_chunk<DT>(x + i, valid);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = (float)c.v[e];
        drop_block(d, (uint32_t)j, v);
        store_chunk<DT>(y + i, valid, v);
    }
}

static __device__ __forceinline__ double block_sum(double v, double *lds) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0;
    for (int k = 0; k < (int)blockDim.x / 64; k++) s += lds[k];
    return s;
}

static __device__ __forceinline__ float activate(float z, int act) {
    if (act == PLENREG_ACT_RELU) return z <= 0.f ? 0.f : z;               // (a NaN stays one)
    if (act == PLENREG_ACT_SILU) return z / (1.f + expf(-z));
    return z;
}
// derivative of the activation at z
static __device__ __forceinline__ float slope(double z, int act) {
    if (act == PLENREG_ACT_RELU) return z > 0 ? 1.f : 0.f;
    if (act == PLENREG_ACT_SILU) { const float s = 1.f / (1.f + expf(-(float)z)); return s * (1.f + (float)z * (1.f - s)); }
    return 1.f;
}

// element l, c of group g of slab n after dropout
template <int DT> static __device__ __forceinline__ double element(const PlenRegNorm &A, const Draw &d, int64_t n, int64_t l, int c, bool &keep) {
    typedef typename Elem<DT>::T T;
    const double v = (double)(float)((const T *)A.x)[n * A.x_stride + l * A.C + c];
    keep = A.cut == 0 || kept(d, (n * A.L + l) * A.C + c);
    return !keep ? 0.0 : A.cut ? v * (65536.0 / (65536.0 - (double)A.cut)) : v;
}

// one workgroup per (n, group): mean, centred squares, result
template <int DT> __global__ __launch_bounds__(256) void k_norm_forward(PlenRegNorm A) {
    typedef typename Elem<DT>::T T;
    __shared__ double lds[4];
    const int D = A.C / A.G, g = blockIdx.x % A.G;
    const int64_t n = blockIdx.x / A.G, count = A.L * D;
    Draw d = {};
    if (A.cut) {
        d = make_draw(A.rng, A.site, A.cut);
        if (A.used && blockIdx.x == 0 && threadIdx.x == 0) { A.used[0] = A.rng[0]; A.used[1] = A.rng[1]; }
    }
    bool keep;
    double s = 0;
    for (int64_t e = threadIdx.x; e < count; e += 256) s += element<DT>(A, d, n, e / D, g * D + (int)(e % D), keep);
    const double mean = block_sum(s, lds) / count;
    s = 0;
    for (int64_t e = threadIdx.x; e < count; e += 256) { const double v = element<DT>(A, d, n, e / D, g * D + (int)(e % D), keep) - mean; s += v * v; }
    const double rstd = 1.0 / sqrt(block_sum(s, lds) / count + (double)A.eps);
    if (A.stats && threadIdx.x == 0) { A.stats[2 * (n * A.G + g)] = mean; A.stats[2 * (n * A.G + g) + 1] = rstd; }
    for (int64_t e = threadIdx.x; e < count; e += 256) {
        const int64_t l = e / D; const int c = g * D + (int)(e % D);
        const float xh = (float)((element<DT>(A, d, n, l, c, keep) - mean) * rstd);
        const float z = xh * load_param(A.w, A.w_dtype, c, 1.f) + load_param(A.b, A.w_dtype, c, 0.f);
        ((T *)A.out)[(n * A.L + l) * A.C + c] = (T)activate(z, A.act);
    }
}

// dz and xh of one element
template <int DT> static __device__ __forceinline__ void gradients(const PlenRegNorm &A, const Draw &d, int64_t n, int64_t l, int c, bool &keep, float &dz, float &xh) {
    typedef typename Elem<DT>::T T;
    const double *st = A.stats + 2 * (n * A.G + c / (A.C / A.G));
    const double h = (element<DT>(A, d, n, l, c, keep) - st[0]) * st[1];
    const double z = h * (double)load_param(A.w, A.w_dtype, c, 1.f) + (double)load_param(A.b, A.w_dtype, c, 0.f);
    xh = (float)h;
    dz = (float)((const T *)A.dy)[n * A.dy_stride + l * A.C + c] * slope(z, A.act);
}
template <int DT> __global__ __launch_bounds__(256) void k_norm_backward(PlenRegNorm A) {
    typedef typename Elem<DT>::T T;
    __shared__ double lds[4];
    const int D = A.C / A.G, g = blockIdx.x % A.G;
    const int64_t n = blockIdx.x / A.G, count = A.L * D;
    Draw d = {};
    if (A.cut) d = make_draw(A.rng, A.site, A.cut);
    bool keep; float dz, xh;
    double s1 = 0, s2 = 0;
    for (int64_t e = threadIdx.x; e < count; e += 256) {
        const int c = g * D + (int)(e % D);
        gradients<DT>(A, d, n, e / D, c, keep, dz, xh);
        const float gw = dz * load_param(A.w, A.w_dtype, c, 1.f);
        s1 += gw; s2 += (double)gw * xh;
    }
    const float m1 = (float)(block_sum(s1, lds) / count), m2 = (float)(block_sum(s2, lds) / count), rstd = (float)A.stats[2 * (n * A.G + g) + 1];
    for (int64_t e = threadIdx.x; e < count; e += 256) {
        const int64_t l = e / D; const int c = g * D + (int)(e % D);
        gradients<DT>(A, d, n, l, c, keep, dz, xh);
        const float v = rstd * (dz * load_param(A.w, A.w_dtype, c, 1.f) - m1 - xh * m2);
        ((T *)A.out)[(n * A.L + l) * A.C + c] = (T)(!keep ? 0.f : A.cut ? v * d.scale : v);
    }
}
// one workgroup per channel: dw, db
template <int DT> __global__ __launch_bounds__(256) void k_norm_params(PlenRegNorm A) {
    __shared__ double lds[4];
    const int c = blockIdx.x;
    Draw d = {};
    if (A.cut) d = make_draw(A.rng, A.site, A.cut);
    bool keep; float dz, xh;
    double s1 = 0, s2 = 0;
    for (int64_t e = threadIdx.x; e < A.N * A.L; e += 256) {
        gradients<DT>(A, d, e / A.L, e % A.L, c, keep, dz, xh);
        s1 += dz; s2 += (double)dz * xh;
    }
    s1 = block_sum(s1, lds); s2 = block_sum(s2, lds);
    if (threadIdx.x == 0) {
        if (A.db) store_param(A.db, A.w_dtype, c, (float)s1);
        if (A.dw) store_param(A.dw, A.w_dtype, c, (float)s2);
    }
}

#define DROPOUT_SMALL (1 << 18)
#define PLENREG_REFUSE (-(int)hipErrorInvalidValue)
#define PLENREG_BY_TYPE(dtype, call)                  \
    switch (dtype) {                                  \
    case PLENREG_F32: call(PLENREG_F32); break;       \
    case PLENREG_BF16: call(PLENREG_BF16); break;     \
    default: call(PLENREG_F16); break;                \
    }

static int launched() { return -(int)hipGetLastError(); }
static bool bad_type(int t) { return t < PLENREG_F32 || t > PLENREG_F16; }
// the mask counts blocks of 8 elements in 32 bits
static bool bad_draw(const uint64_t *rng, uint32_t cut, int site, int64_t n) { return cut > 65536u || site < 0 || (cut && (!rng || n > ((int64_t)1 << 35))); }
static bool bad_norm(const PlenRegNorm *a) {
    return !a || a->N < 1 || a->L < 1 || a->C < 1 || a->G < 1 || a->C % a->G || a->C > (a->L > 1 ? PLENREG_MAX_C_LONG : PLENREG_MAX_C) || bad_type(a->dtype) || bad_type(a->w_dtype)
           || a->act < PLENREG_ACT_NONE || a->act > PLENREG_ACT_SILU || !(a->eps > 0.f) || a->N > ((int64_t)1 << 31) - 1 || a->L > ((int64_t)1 << 40) / a->C || a->N > ((int64_t)1 << 40) / (a->L * a->C)
           || a->N * (int64_t)a->G > ((int64_t)1 << 31) - 1 || bad_draw(a->cut ? (const uint64_t *)1 : nullptr, a->cut, a->site, a->N * a->L * a->C);
}

extern "C" {

int plenreg_dropout(const PlenRegDropout *a, void *stream) {
    if (!a || !a->x || !a->y || !a->rng || a->rows < 1 || a->cols < 1 || a->rows > ((int64_t)1 << 35) / a->cols || a->x_stride < 0 || bad_type(a->dtype)
        || bad_draw(a->rng, a->cut, a->site, a->rows * a->cols)) return PLENREG_REFUSE;
    const int64_t chunks = (a->rows * a->cols + 7) / 8;
    const bool rows = a->rows > 1 && a->x_stride != a->cols, small = chunks <= DROPOUT_SMALL;
    const dim3 grid((unsigned)((chunks + (small ? 255 : 1023)) / (small ? 256 : 1024)));
#define CALL(DT)                                                                                                                              \
    small ? (rows ? k_dropout<DT, 1, true><<<grid, 256, 0, (hipStream_t)stream>>>(*a) : k_dropout<DT, 1, false><<<grid, 256, 0, (hipStream_t)stream>>>(*a)) \
          : (rows ? k_dropout<DT, 4, true><<<grid, 256, 0, (hipStream_t)stream>>>(*a) : k_dropout<DT, 4, false><<<grid, 256, 0, (hipStream_t)stream>>>(*a))
    PLENREG_BY_TYPE(a->dtype, CALL)
#undef CALL
    return launched();
}

int64_t plenreg_norm_workspace(const PlenRegNorm *a, int backward) {
    (void)backward;
    return bad_norm(a) ? PLENREG_REFUSE : 0;
}

int plenreg_norm_forward(const PlenRegNorm *a, void *stream) {
    if (bad_norm(a) || !a->x || !a->out || a->x_stride < 0 || (a->cut && !a->rng)) return PLENREG_REFUSE;
    const dim3 grid((unsigned)(a->N * a->G));
#define CALL(DT) k_norm_forward<DT><<<grid, 256, 0, (hipStream_t)stream>>>(*a)
    PLENREG_BY_TYPE(a->dtype, CALL)
#undef CALL
    return launched();
}

int plenreg_norm_backward(const PlenRegNorm *a, void *stream) {
    if (bad_norm(a) || !a->x || !a->dy || !a->out || !a->stats || a->x_stride < 0 || a->dy_stride < 0 || (a->cut && !a->rng)) return PLENREG_REFUSE;
    const dim3 grid((unsigned)(a->N * a->G));
#define CALL(DT) k_norm_backward<DT><<<grid, 256, 0, (hipStream_t)stream>>>(*a)
    PLENREG_BY_TYPE(a->dtype, CALL)
#undef CALL
    if (a->dw || a->db) {
        const dim3 cols((unsigned)a->C);
#define CALL(DT) k_norm_params<DT><<<cols, 256, 0, (hipStream_t)stream>>>(*a)
        PLENREG_BY_TYPE(a->dtype, CALL)
#undef CALL
    }
    return launched();
}

const char *plenreg_version(void) { return "libplenreg 1.0 gfx950"; }

}  // extern "C"
