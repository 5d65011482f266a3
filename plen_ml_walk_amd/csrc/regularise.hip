// regularise.hip -- the C ABI of include/plenreg.h (argument checks, launch plans) and the dropout kernel; the group-norm kernels are in regularise_norm.hip.
// Small calls are bound by launch latency, dropout and long slabs by memory traffic, wide layers with dropout and SiLU by vector issue.
#include "regularise.h"

#define DROPOUT_SMALL (1 << 18)
#define STREAM_BYTES ((int64_t)64 << 20)     // last readings and results of tensors from here on go past the caches (2 x 262144 x 128 bf16, passes back to back: sums 47 -> 26 us, since no results of the pass
                                             // before have to be written back meanwhile; result 42 -> 40.  By size alone: what a later reader of the result pays was not measured)
#define MAP_MAX_SPAN ((int64_t)1 << 28)      // elements of a slab that one workgroup walks over
#define ROW_MAX 8192                    // widest group that the lanes of one workgroup hold: 256 lanes of 4 chunks, or in the backward pass (which holds four times as much) 512 of one or two

// ---- dropout.  U chunks per thread: all loads are issued before the first mask is drawn.  In rows that are not contiguous (ROWS) a chunk that crosses
//      the end of a row is loaded element by element.  Memory: 32768 x 4096 bf16 77 us = 7.0 TB/s read and written, with the reads past the caches (92 with them in the caches; with the
//      writes past them too the kernel alone is slower).  100 x 256 f32 2.3 us: the launch.
struct DropArgs { const void *x; void *y; const uint64_t *rng; uint64_t *used; int64_t rows, cols, x_stride; uint32_t cut; int site; float scale; };
template <int DT, int U, bool ROWS> __global__ __launch_bounds__(256) void k_dropout(DropArgs A) {
    typedef typename Elem<DT>::T T;
    const T *x = (const T *)A.x;
    T *y = (T *)A.y;
    const Draw d = make_draw(A.rng, A.site, A.cut);
    if (A.used && blockIdx.x == 0 && threadIdx.x == 0) { A.used[0] = A.rng[0]; A.used[1] = A.rng[1]; }
    const int64_t n = A.rows * A.cols, first = (int64_t)blockIdx.x * (256 * U);
    if (!ROWS && (first + 256 * U) * 8 <= n) {                     // every chunk of the workgroup is whole
        Chunk<DT> c[U];
#pragma unroll
        for (int u = 0; u < U; u++) c[u] = U > 1 ? stream_whole<DT>(x + (first + u * 256 + threadIdx.x) * 8) : load_whole<DT>(x + (first + u * 256 + threadIdx.x) * 8);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const Mask<2> m(d, (first + u * 256 + threadIdx.x) * 8);
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = m.keep(e, c[u].get(e) * A.scale);
            store_whole<DT>(y + (first + u * 256 + threadIdx.x) * 8, v);
        }
        return;
    }
    for (int u = 0; u < U; u++) {
        const int64_t j = first + u * 256 + threadIdx.x, i = j << 3;
        if (i >= n) return;
        const int valid = n - i < 8 ? (int)(n - i) : 8;
        float v[8];
        int64_t row = 0, col = i;
        if (ROWS) {
            row = n >> 32 ? i / A.cols : (int64_t)((uint32_t)i / (uint32_t)A.cols);
            col = i - row * A.cols;
        }
        if (!ROWS || col + valid <= A.cols) {
            const Chunk<DT> c = load_chunk<DT>(x + row * A.x_stride + col, valid);
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = c.get(e);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                v[e] = e < valid ? (float)x[row * A.x_stride + col] : 0.f;
                if (++col == A.cols) { col = 0; row++; }
            }
        }
        const Mask<2> m(d, i);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = m.keep(e, v[e] * A.scale);
        store_chunk<DT>(y + i, valid, v);
    }
}

// ---- argument checks
#define PLENREG_REFUSE (-(int)hipErrorInvalidValue)
static int launched() { return -(int)hipGetLastError(); }
static bool bad_type(int t) { return t < PLENREG_F32 || t > PLENREG_F16; }
// the mask counts blocks of 8 elements in 32 bits
static bool bad_draw(uint32_t cut, int site, int64_t n) { return cut > 65536u || site < 0 || (cut && n > ((int64_t)1 << 35)); }
static bool bad_norm(const PlenRegNorm *a) {
    return !a || a->N < 1 || a->L < 1 || a->C < 1 || a->G < 1 || a->C % a->G || a->C > (a->L > 1 ? PLENREG_MAX_C_LONG : PLENREG_MAX_C) || bad_type(a->dtype)
           || (a->w_dtype != PLENREG_F32 && a->w_dtype != a->dtype) || a->act < PLENREG_ACT_NONE || a->act > PLENREG_ACT_SILU || !(a->eps > 0.f) || a->N > ((int64_t)1 << 31) - 1
           || a->L > ((int64_t)1 << 40) / a->C || a->N > ((int64_t)1 << 40) / (a->L * a->C) || a->N * (int64_t)a->G > ((int64_t)1 << 31) - 1 || bad_draw(a->cut, a->site, a->N * a->L * a->C);
}
static double drop_scale(uint32_t cut) { return cut < 65536u ? 65536.0 / (65536.0 - (double)cut) : 0.0; }

// ---- launch plans: functions of the sizes alone, so that a workspace asked for and the launch that uses it agree
static int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }
static int log2_up(int64_t v) { int k = 0; while (((int64_t)1 << k) < v) k++; return k; }

static bool by_rows(const PlenRegNorm &a) { return a.L == 1 && a.C / a.G <= ROW_MAX; }
// is a tensor of x's shape beyond what the caches keep?
static bool streams(const PlenRegNorm &a) { return a.N * a.L * a.C * (a.dtype == PLENREG_F32 ? 4 : 2) >= STREAM_BYTES; }
static RowLaunch row_plan(const PlenRegNorm &a, bool backward) {
    const int64_t chunks = div_up(a.C / a.G, 8);
    RowLaunch r;
    // forward: up to 4 chunks per lane, so that rows of up to 2048 elements need no barrier; backward: one while 512 lanes are enough (us, one / two chunks, bf16: 16384 x 4096 92 / 104,
    // 16384 x 2048 49 / 59; f32 177 / 203, 89 / 108)
    r.K = backward ? (chunks <= 512 ? 1 : 2) : chunks <= 64 ? 1 : chunks <= 128 ? 2 : 4;
    r.NT = backward ? 512 : 256;
    r.P.team_log = log2_up(div_up(chunks, r.K));
    const int teams = r.NT >> r.P.team_log;
    r.P.gb = a.G < teams ? a.G : teams;
    r.P.inv_gb = 1.f / (float)r.P.gb;
    r.P.rb = teams / r.P.gb;
    const int64_t gy = div_up(a.G, r.P.gb), need = div_up(a.N, r.P.rb);
    // as many workgroups as are resident at a time, each over several rows; in the backward pass at most 256 rows per lane (its 32-bit sums)
    int64_t gx = div_up(backward ? 512 : r.K == 4 ? 512 : 1024, gy);
    if (backward && gx < div_up(need, 256)) gx = div_up(need, 256);
    if (gx > need) gx = need;
    r.P.trips = (int)div_up(need, gx);
    r.grid = dim3((unsigned)gx, (unsigned)gy);
    r.stream = streams(a);
    return r;
}
static WideLaunch wide_plan(const PlenRegNorm &a) {
    WideLaunch m;
    m.grid = (unsigned)(a.N * a.G < 2048 ? a.N * a.G : 2048);
    // parameter gradients: about 1024 workgroups, of at least 8 rows (each leaves 2 C partial sums) and at most 256 (their sums are in 32 bits)
    const int64_t x = div_up((int64_t)a.G * div_up(a.C / a.G, 8), 256);
    int64_t y = div_up(1024, x);
    if (y > div_up(a.N, 8)) y = div_up(a.N, 8);
    if (y < div_up(a.N, 256)) y = div_up(a.N, 256);
    if (y > a.N) y = a.N;
    m.params = dim3((unsigned)x, (unsigned)(y < 65535 ? y : 65535));
    m.stream = streams(a);
    return m;
}
// threads (a multiple of 64) of which the fewest idle when `ncol` of them make a row
static int fill_threads(int ncol, int lo, int hi) {
    int best = lo;
    double most = 0.0;
    for (int nt = lo; nt <= hi; nt += 64) {
        const double used = (double)(nt / ncol * ncol) / nt;
        if (used > most + 1e-9) { most = used; best = nt; }
    }
    return best;
}
// log of a power of two of lanes: at most `there`, one wave's, and no more than there are entries
static int lanes_for(int there, int entries) {
    int log = 0;
    while (log < 6 && 2 << log <= there && 1 << log < entries) log++;
    return log;
}
static MapLaunch map_plan(const PlenRegNorm &a, bool backward) {
    MapLaunch m;
    const int D = a.C / a.G;
    const int64_t size = a.L * a.C;
    m.P.q_log = 0;
    while (((int64_t)a.C << m.P.q_log) % 8) m.P.q_log++;
    const int64_t columns = ((int64_t)a.C << m.P.q_log) / 8, chunks = div_up(size, 8);
    m.P.ncol = (int)(columns < chunks ? columns : chunks);
    m.P.rows = div_up(a.L, (int64_t)1 << m.P.q_log);
    m.P.col_blocks = (int)div_up(m.P.ncol, 512);
    m.P.bcol = (int)div_up(m.P.ncol, m.P.col_blocks);
    m.P.inv_bcol = 1.f / (float)m.P.bcol;
    // one workgroup per slab: one launch instead of two or three, and the slab is read once from memory; but only as many compute units work as there are slabs, and nothing goes past
    // the caches.  Measured (us, slab / split; N x L x C bf16; before each group had its own shift, which costs both forms 1-5 %): forward 8 x 32 x 320 6.3 / 8.2, 8 x 128 x 195 8.1 / 8.5, 8 x 1024 x 32 7.5 / 6.7, 64 x 128 x 320 10.8 / 11.0, 64 x 512 x 128
    // 12.4 / 9.5, 256 x 128 x 320 13.6 / 16.5, 256 x 512 x 320 42.9 / 44.2, 2048 x 64 x 320 47 / 53, 20000 x 16 x 64 32 / 77, beyond what the caches hold 1024 x 512 x 320 203 / 170,
    // 8192 x 256 x 64 145 / 132.  Backward, groups that share chunks: 8 x 32 x 320 14.0 / 13.7, 64 x 128 x 195 26.7 / 23.4, 256 x 32 x 320 16.4 / 27.8, 256 x 512 x 320 77 / 123, 1024 x 512 x 320
    // 329 / 418; groups of whole chunks: 256 x 512 x 128 38.1 / 35.9, 2048 x 256 x 64 91 / 67, 20000 x 49 x 96 522 / 454, 20000 x 16 x 64 106 / 164.
    const bool whole = a.C % 8 == 0 && D % 8 == 0, many = a.N >= 256 && size <= 262144;
    m.slab = m.P.bcol <= 448 && m.P.col_blocks == 1 && a.G <= 512
             && (backward ? size <= (whole ? 4096 : 8192) || (many && !whole)
                          : size <= 4096 || ((size <= 25600 || (a.N >= 64 && size <= 40960) || many) && a.N * size * (a.dtype == PLENREG_F32 ? 4 : 2) < (int64_t)192 << 20));
    const int64_t threads = div_up(chunks, 64) * 64;
    m.NT = m.slab ? fill_threads(m.P.bcol, threads < 448 ? (int)threads : 448, 448) : fill_threads(m.P.bcol, 256, 512);
    m.P.R = m.NT / m.P.bcol;
    // 2 workgroups per compute unit, or 4 where their threads then still have 16 chunks each; each thread in whole turns of 2 rows.  One, where their joins weigh more than their number
    // helps: a slab with more than 2048 partial pairs, and the backward pass of groups that share chunks.  (us; 512 / 256 / 1024 workgroups: 8 x 4096 x 320 forward 17.0 / 18.3 / 19.5,
    // backward 42.4 / 35.6 / 56.9; 1 x 4096 x 512 in 8 groups 9.0 / 8.1 / 9.0 and 16.6 / 14.2 / 16.2; 2 x 16384 x 128 in 8 groups 9.8 / 10.1 / 12.0 and 16.6 / 18.5 / 20.9; 2 x 262144 x 128
    // sums 47 with 512, 40 with 1024)
    const int64_t groups = a.N * m.P.col_blocks;
    int64_t blocks = a.N * chunks >= (int64_t)1 << 22 ? 1024 : 512;
    if (blocks == 512 && ((backward && !whole) || div_up(512, groups) * a.G * m.P.col_blocks > 2048)) blocks = 256;
    const int64_t turn = (int64_t)m.P.R * 2, turns = div_up(m.P.rows, turn);
    const int64_t most = MAP_MAX_SPAN / (turn * ((int64_t)a.C << m.P.q_log));              // turns of a workgroup, so that its offsets fit
    const int64_t per = div_up(turns, groups >= blocks ? 1 : div_up(blocks, groups));
    m.P.rows_per = m.P.apply_rows = (per < most ? per : most) * turn;
    m.P.splits = (int)div_up(m.P.rows, m.P.rows_per);
    const int64_t row_blocks = div_up(m.P.rows, m.P.apply_rows);
    // lanes that join a group (a channel) of a workgroup's entries: all of them at a time where there are as many
    const int units = whole ? D / 8 : D >= 8 ? (D + 14) / 8 : D, local = (int)(m.P.q_log || m.P.bcol * 8 > a.C ? a.C : m.P.bcol * 8);
    m.P.lanes_log = lanes_for(m.NT / a.G, (units * m.P.R) << m.P.q_log);
    m.P.chan_log = lanes_for(m.NT / local, m.P.R << m.P.q_log);
    // slabs beyond what fills the chip (and the grid's limit of 65535) are walked by the workgroups
    int64_t z = div_up(2048, m.P.splits);
    m.sums = dim3((unsigned)m.P.splits, (unsigned)m.P.col_blocks, (unsigned)(a.N < z ? a.N : z));
    m.param_rows = (int)(m.sums.x * (m.P.q_log ? m.sums.y : 1) * m.sums.z);
    z = div_up(8192, row_blocks);
    m.apply = dim3((unsigned)row_blocks, (unsigned)m.P.col_blocks, (unsigned)(a.N < z ? a.N : z));
    if (m.slab) {
        m.P.rows_per = m.P.rows; m.P.splits = 1;
        m.sums = dim3(1, (unsigned)(a.N < 2048 ? a.N : 2048), 1);
        m.param_rows = (int)m.sums.y;
    }
    m.lean = (int64_t)m.sums.x * m.sums.y * m.sums.z > 512;
    m.walks = a.N > (m.slab ? m.sums.y : m.sums.z);
    // few partial pairs per slab: every workgroup of the result's launch joins them for itself (32 KB out of the caches at 2048 pairs), and there is no launch between.
    // Measured (us, so / with a launch of its own; bf16, pairs per slab): forward 8 x 4096 x 320 2048 18.4 / 19.5, 4096 19.1 / 19.4, 10240 22.5 / 19.5, 2 x 16384 x 128 2048 9.9 / 11.4,
    // 1 x 4096 x 512 16384 13.1 / 11.3; both passes 4 x 1089 x 195 455 36.4 / 38.5, 2275 37.2 / 39.0, 8 x 4096 x 320 2048 65.5 / 66.4, 4096 67.8 / 66.7
    m.joins = (int64_t)a.G * m.P.splits * m.P.col_blocks <= (backward ? 2560 : 4096);
    m.P.param_z = 0;
    m.P.join_log = lanes_for(m.NT / a.G, 64);
    m.stream = streams(a);
    m.stat_blocks = (unsigned)(a.N * a.G < 4 * 65536 ? div_up(a.N * a.G, 4) : 65536);
    return m;
}
// bytes of a map launch's parameter sums: a row of 2 C per workgroup, and where it walks over slabs the same in 64 bits in front of them
static int64_t sums_bytes(const PlenRegNorm &a, const MapLaunch &m) { return (int64_t)m.param_rows * 2 * a.C * (m.walks ? 12 : 4); }
// bytes of the partial pairs of a map launch
static int64_t part_bytes(const PlenRegNorm &a, const MapLaunch &m) { return a.N * a.G * m.P.splits * m.P.col_blocks * 16; }

static const NormEntry &entry(const PlenRegNorm &a) {
    if (a.dtype == PLENREG_F32) return plenreg_norm_f32_f32();
    if (a.dtype == PLENREG_BF16) return a.w_dtype == PLENREG_F32 ? plenreg_norm_bf16_f32() : plenreg_norm_bf16_bf16();
    return a.w_dtype == PLENREG_F32 ? plenreg_norm_f16_f32() : plenreg_norm_f16_f16();
}
static NormArgs kernel_args(const PlenRegNorm &a) {
    NormArgs k;
    k.x = a.x; k.dy = a.dy; k.w = a.w; k.b = a.b; k.out = a.out; k.stats = (double2 *)a.stats; k.rng = a.rng; k.used = a.used;
    k.N = a.N; k.x_stride = a.x_stride; k.dy_stride = a.dy_stride; k.size = a.L * a.C;
    k.C = a.C; k.G = a.G; k.D = a.C / a.G; k.act = a.act; k.site = a.site; k.cut = a.cut;
    k.count = (double)a.L * k.D; k.inv_count = 1.0 / k.count; k.scale = drop_scale(a.cut); k.eps = (double)a.eps;
    k.inv_D = 1.f / (float)k.D; k.inv_C = 1.f / (float)a.C;
    return k;
}

extern "C" {

int plenreg_dropout(const PlenRegDropout *a, void *stream) {
    if (!a || !a->x || !a->y || !a->rng || a->rows < 1 || a->cols < 1 || a->rows > ((int64_t)1 << 35) / a->cols || a->x_stride < 0 || bad_type(a->dtype) || bad_draw(a->cut, a->site, a->rows * a->cols))
        return PLENREG_REFUSE;
    const DropArgs k = {a->x, a->y, a->rng, a->used, a->rows, a->cols, a->x_stride, a->cut, a->site, (float)drop_scale(a->cut)};
    const hipStream_t s = (hipStream_t)stream;
    // few chunks: one per thread, so that every compute unit gets some; many: four, whose loads are in flight together
    const int64_t chunks = div_up(a->rows * a->cols, 8);
    const bool rows = a->rows > 1 && a->x_stride != a->cols, small = chunks <= DROPOUT_SMALL;
    const unsigned grid = (unsigned)div_up(chunks, small ? 256 : 1024);
#define CALL(DT)                                                                                          \
    if (small) { if (rows) k_dropout<DT, 1, true><<<grid, 256, 0, s>>>(k); else k_dropout<DT, 1, false><<<grid, 256, 0, s>>>(k); } \
    else if (rows) k_dropout<DT, 4, true><<<grid, 256, 0, s>>>(k);                                        \
    else k_dropout<DT, 4, false><<<grid, 256, 0, s>>>(k)
    if (a->dtype == PLENREG_F32) { CALL(PLENREG_F32); }
    else if (a->dtype == PLENREG_BF16) { CALL(PLENREG_BF16); }
    else { CALL(PLENREG_F16); }
#undef CALL
    return launched();
}

int64_t plenreg_norm_workspace(const PlenRegNorm *a, int backward) {
    if (bad_norm(a)) return PLENREG_REFUSE;
    if (by_rows(*a)) return backward ? (int64_t)row_plan(*a, true).grid.x * 2 * a->C * 4 : 0;
    if (a->L == 1) return backward ? (int64_t)wide_plan(*a).params.y * 2 * a->C * 4 : 0;
    const MapLaunch m = map_plan(*a, backward);
    if (m.slab) return backward ? sums_bytes(*a, m) : 0;
    return part_bytes(*a, m) + a->N * a->G * 16 + (backward ? sums_bytes(*a, m) : 0);
}

int plenreg_norm_forward(const PlenRegNorm *a, void *stream) {
    if (bad_norm(a) || !a->x || !a->out || a->x_stride < 0 || (a->cut && !a->rng)) return PLENREG_REFUSE;
    NormArgs k = kernel_args(*a);
    if (by_rows(*a)) {
        entry(*a).row_forward(k, row_plan(*a, false), (hipStream_t)stream);
        return launched();
    }
    if (a->L == 1) {
        entry(*a).wide_forward(k, wide_plan(*a), (hipStream_t)stream);
        return launched();
    }
    const MapLaunch m = map_plan(*a, false);
    if (!a->ws && !m.slab) return PLENREG_REFUSE;
    if (!k.stats && !m.slab) k.stats = (double2 *)((char *)a->ws + part_bytes(*a, m));
    entry(*a).map_forward(k, m, (double2 *)a->ws, (hipStream_t)stream);
    return launched();
}

int plenreg_norm_backward(const PlenRegNorm *a, void *stream) {
    if (bad_norm(a) || !a->x || !a->dy || !a->out || !a->stats || a->x_stride < 0 || a->dy_stride < 0 || (a->cut && !a->rng)) return PLENREG_REFUSE;
    const bool params = a->dw || a->db, rows = by_rows(*a);
    if (plenreg_norm_workspace(a, 1) > 0 && (params || a->L > 1) && !a->ws) return PLENREG_REFUSE;
    const NormArgs k = kernel_args(*a);
    const NormEntry &e = entry(*a);
    if (rows) {
        const RowLaunch r = row_plan(*a, true);
        e.row_backward(k, r, params ? (float *)a->ws : nullptr, (hipStream_t)stream);
        if (params) e.params(k, (const float *)a->ws, (int)r.grid.x, a->dw, a->db, (hipStream_t)stream);
        return launched();
    }
    if (a->L == 1) {
        const WideLaunch m = wide_plan(*a);
        e.wide_backward(k, m, params ? (float *)a->ws : nullptr, (hipStream_t)stream);
        if (params) e.params(k, (const float *)a->ws, (int)m.params.y, a->dw, a->db, (hipStream_t)stream);
        return launched();
    }
    const MapLaunch m = map_plan(*a, true);
    char *ws = (char *)a->ws;
    double2 *means = (double2 *)(ws + part_bytes(*a, m));
    double *running = !params ? nullptr : m.slab ? (double *)ws : (double *)(means + a->N * a->G);
    float *sums = (float *)(running && m.walks ? running + (int64_t)m.param_rows * 2 * a->C : running);
    e.map_backward(k, m, (double2 *)ws, means, sums, running, a->dw, a->db, (hipStream_t)stream);
    return launched();
}

const char *plenreg_version(void) { return "libplenreg 1.0 gfx950"; }

}  // extern "C"
