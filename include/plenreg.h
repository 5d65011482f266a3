/*
 * plenreg.h -- C ABI of libplenreg.so: the regularisation operators of the Q networks' hidden layers as hand-written HIP kernels (gfx950):
 * dropout whose mask is drawn from the counter-based generator and never stored, group norm with an activation over channels-last data,
 * and the two in one pass, each with its gradient.  plen_ml_walk_amd/regularise.py loads the library and hands its entry points to the autograd nodes of
 * csrc/regularise_torch.cpp, which call them.
 *
 * Conventions: every pointer is a caller-owned DEVICE pointer; work is enqueued on the hipStream_t passed as `stream` and is capturable in a
 * hipGraph; nothing is allocated and no state is kept between calls.  Outputs overlap neither inputs nor each other.  Return 0, or a negative HIP error code (-1 = hipErrorInvalidValue:
 * an argument is outside what this header allows; nothing was launched then).
 */
#ifndef PLENREG_H
#define PLENREG_H
#include <stdint.h>
#ifdef __cplusplus
extern "C" {
#endif

/* element types of x, dy, y, dx and of the parameters */
#define PLENREG_F32 0
#define PLENREG_BF16 1
#define PLENREG_F16 2
/* activations */
#define PLENREG_ACT_NONE 0
#define PLENREG_ACT_RELU 1
#define PLENREG_ACT_SILU 2

/* The mask.  rng = device uint64[2] {seed, calls so far} (the state of every draw of this package: Philox4x32-10).  Element i of a tensor, counted
 * row-major over its logical shape, takes the 16-bit half number (i & 7), low half first, of the words philox(counter = (i >> 3, calls lo, calls hi,
 * 16 + site), key = seed); it is kept where that half is >= cut, i.e. it is dropped with probability cut / 65536, and kept values are multiplied by
 * 65536 / (65536 - cut) (0 if cut is 65536: everything is dropped).  cut = 0: no dropout.  `used` (or NULL) receives {seed, calls} as the kernel
 * read them, 16 bytes from which the backward pass draws the same mask again after the state has moved on; the state itself is not advanced. */

typedef struct PlenRegDropout {
    const void *x;             /* [rows][cols], consecutive rows x_stride elements apart */
    void *y;                   /* [rows][cols], contiguous */
    const uint64_t *rng;
    uint64_t *used;
    int64_t rows, cols, x_stride;
    int32_t dtype;
    uint32_t cut;              /* 0 .. 65536 */
    int32_t site;              /* >= 0 */
} PlenRegDropout;
/* y = kept ? x scale : 0.  The gradient is the same call on dy, with rng = the forward's `used`. */
int plenreg_dropout(const PlenRegDropout *args, void *stream);

typedef struct PlenRegNorm {
    const void *x;             /* N slabs of L x C contiguous elements, x_stride elements apart */
    const void *dy;            /* backward: likewise, dy_stride apart */
    const void *w, *b;         /* [C] of type w_dtype, which is PLENREG_F32 or dtype; NULL: ones / zeros */
    void *out;                 /* forward: y, backward: dx; [N][L][C] contiguous */
    double *stats;             /* [N][G][2], 16-byte aligned: mean m of the masked but unscaled input and r = scale / sqrt(scale^2 variance + eps), so that the normalised
                                * value is (x - m) r, with dropout or without; written by the forward pass (NULL: not wanted), read by the backward pass */
    void *dw, *db;             /* backward: [C] of type w_dtype, written; NULL: not wanted */
    void *ws;                  /* plenreg_norm_workspace() bytes, 16-byte aligned; contents need not be preserved or cleared */
    const uint64_t *rng;       /* cut > 0 only; backward: the forward's `used` */
    uint64_t *used;            /* forward, cut > 0 only */
    int64_t N, L, x_stride, dy_stride;
    int32_t C, G;              /* G divides C */
    int32_t dtype, w_dtype, act;
    uint32_t cut;
    int32_t site;
    float eps;                 /* > 0 */
} PlenRegNorm;
#define PLENREG_MAX_C 32768            /* widest row with L = 1 */
#define PLENREG_MAX_C_LONG 8192        /* widest row with L > 1 */
/* y = act(((d(x) - mean) rstd) w + b), d = dropout (cut > 0) or the identity; mean and variance over the L x (C / G) elements of each (n, group).  What one group holds (NaN, infinity, any size)
 * changes no other group's results, in either pass. */
int plenreg_norm_forward(const PlenRegNorm *args, void *stream);
/* dx, dw, db of the above from dy, x and stats */
int plenreg_norm_backward(const PlenRegNorm *args, void *stream);
/* bytes of workspace that the forward (backward = 0) / backward (1) pass of these sizes needs; negative: the sizes are not allowed */
int64_t plenreg_norm_workspace(const PlenRegNorm *args, int backward);

const char *plenreg_version(void);

#ifdef __cplusplus
}
#endif
#endif
