// regularise_norm.hip -- group norm with an activation, with dropout before it or without, for one pair of element types: REG_DT of x and of the results, REG_WT of
// the parameters; REG_ENTRY names the table of launches.
//
// Statistics are sums of (x - s) and (x - s)^2 in 64 bits, s = the group's own first element: a 64-bit addition costs a vector slot like a 32-bit one on this chip, one
// pass over the data is enough, the sums of different workgroups join by addition, a constant group has exactly no variance, the variance survives a
// mean of any size, and a group's NaN or infinity stays its own.  (It is also what the gate of ReLU's gradient is decided with.)  The rest is in 32 bits, with the mean as a sum of two floats, so that x - mean is
// exact to a rounding of its own.
//
// Code size counts: the instruction cache is cold at each launch, and a kernel that runs its text once is bound by fetching it.  So: quotients come from the
// host, the form without partial chunks (V > 0) is a variant of its own, parameter types are compiled in.
//
// No variant may spill to scratch memory (tests/test_regularise_cpu.py): a spilling one has lost values of lanes that a divergent branch left out.
#include "regularise.h"

#define DT REG_DT
#define WT REG_WT
typedef Elem<DT>::T T;
typedef Elem<WT>::T W;
// variants V: rows 0 = groups that end within a chunk, 1 = whole chunks; slabs 1 = chunks that span groups, 2 = one group each
namespace {

__device__ __forceinline__ float logistic(float z) {
    // 16-bit results: exponential and reciprocal from the hardware's approximations, off by (|z| + 4) 2^-24 of the value, a 2^8th of the result's own rounding and less
    if (DT != PLENREG_F32) return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.44269504f));
    return 1.f / (1.f + expf(-z));
}
__device__ __forceinline__ void activate(float (&z)[8], int act) {
    if (act == PLENREG_ACT_RELU) {
#pragma unroll
        for (int e = 0; e < 8; e++) z[e] = z[e] <= 0.f ? 0.f : z[e];             // (a NaN stays one)
    } else if (act == PLENREG_ACT_SILU) {
#pragma unroll
        for (int e = 0; e < 8; e++) z[e] *= logistic(z[e]);
    }
}
// 1 / sqrt(v) in 64 bits: the hardware's approximation and two Newton steps
__device__ __forceinline__ double inverse_sqrt(double v) {
    double r = __builtin_amdgcn_rsq(v);
    r = fma(0.5 * r, fma(-v * r, r, 1.0), r);
    return fma(0.5 * r, fma(-v * r, r, 1.0), r);
}
// sums of (x - s), (x - s)^2 -> the pair that NormArgs.stats holds
__device__ __forceinline__ double2 finish_stats(const NormArgs &A, double count, double s, double sum, double squares) {
    double m = sum * A.inv_count;
    m = fma(fma(-m, count, sum), A.inv_count, m);          // the quotient to its last bit: an element that is exactly the mean has z = 0, and without a bias a shut gate
    double var = fma(-m, m, squares * A.inv_count);
    if (var < 0.0) var = 0.0;
    return double2{s + m, A.scale * inverse_sqrt(fma(var, A.scale * A.scale, A.eps))};
}
// The normalised value with the mean in two words, mean + rest: (v - mean) rstd + offset, offset = -rest rstd once per group.  The first word alone is off by up to 2^-25 of the mean, which may be far
// above the spread, in 16-bit types too: of 8000 elements around 1000, three of them a step higher, the others are half a percent off.
__device__ __forceinline__ float from_mean(float v, float mean, float rstd, float offset) { return fmaf(v - mean, rstd, offset); }
__device__ __forceinline__ void write_used(const NormArgs &A) {
    if (A.used && blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0 && threadIdx.x == 0) { A.used[0] = A.rng[0]; A.used[1] = A.rng[1]; }
}
// a chunk's elements as floats
template <int E> __device__ __forceinline__ void unpack(const Chunk<E> &c, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = c.get(e);
}
// ... masked ones as zeros
template <int E, int M> __device__ __forceinline__ void unpack(const Chunk<E> &c, const Mask<M> &m, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = m.keep(e, c.get(e));
}

// ---- loads without branches.  A load under a condition waits for the ones before it, so every lane loads whole chunks from inside its row or slab of `size` elements, and
//      what is not asked for is left out of the sums and not stored.  V = 0: the last chunk of a row may begin less than 8 elements before its end: then the 8 last elements are
//      loaded and moved down.
template <int V, int E, bool STREAM = false> __device__ __forceinline__ Chunk<E> load_inside(const typename Elem<E>::T *p, int64_t off, int64_t size) {
    if (V) return STREAM ? stream_whole<E>(p + off) : load_whole<E>(p + off);
    if (size < 8) return load_chunk<E>(p + off, (int)(size - off));
    return load_whole<E>(p + (off < size - 8 ? off : size - 8));
}
template <int V> __device__ __forceinline__ void move_down(float (&v)[8], int64_t off, int64_t size) {
    if (V || size < 8 || off <= size - 8) return;
    const int by = (int)(off - (size - 8));
    if (by & 4) {
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = v[e + 4];
    }
    if (by & 2) {
#pragma unroll
        for (int e = 0; e < 6; e++) v[e] = v[e + 2];
    }
    if (by & 1) {
#pragma unroll
        for (int e = 0; e < 7; e++) v[e] = v[e + 1];
    }
}

// ---- sums over 2^log neighbouring lanes, left in each of them: exchanges within 16 lanes by DPP, beyond by the row swaps
template <int CTRL> __device__ __forceinline__ float from_lane(float v) { return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true)); }
template <int CTRL> __device__ __forceinline__ double from_lane(double v) {
    const int lo = __builtin_amdgcn_mov_dpp(__double2loint(v), CTRL, 0xf, 0xf, true), hi = __builtin_amdgcn_mov_dpp(__double2hiint(v), CTRL, 0xf, 0xf, true);
    return __hiloint2double(hi, lo);
}
// v of this row of 16 (half of 32) lanes + v of its neighbour
__device__ __forceinline__ float add_swapped(float v, bool halves) {
    const uint32_t u = __float_as_uint(v);
    const auto s = halves ? __builtin_amdgcn_permlane32_swap(u, u, false, false) : __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}
__device__ __forceinline__ double add_swapped(double v, bool halves) {
    const uint32_t lo = (uint32_t)__double2loint(v), hi = (uint32_t)__double2hiint(v);
    const auto a = halves ? __builtin_amdgcn_permlane32_swap(lo, lo, false, false) : __builtin_amdgcn_permlane16_swap(lo, lo, false, false);
    const auto b = halves ? __builtin_amdgcn_permlane32_swap(hi, hi, false, false) : __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
    return __hiloint2double((int)b[0], (int)a[0]) + __hiloint2double((int)b[1], (int)a[1]);
}
template <typename F> __device__ __forceinline__ void lanes_sum2(F &a, F &b, int log) {
    if (log < 1) return;
    a += from_lane<0xB1>(a); b += from_lane<0xB1>(b);            // lane ^ 1
    if (log < 2) return;
    a += from_lane<0x4E>(a); b += from_lane<0x4E>(b);            // lane ^ 2
    if (log < 3) return;
    a += from_lane<0x141>(a); b += from_lane<0x141>(b);          // mirrored in 8 lanes (all four lanes of each half hold the same by now)
    if (log < 4) return;
    a += from_lane<0x140>(a); b += from_lane<0x140>(b);          // mirrored in 16 lanes
    if (log < 5) return;
    a = add_swapped(a, false); b = add_swapped(b, false);
    if (log < 6) return;
    a = add_swapped(a, true); b = add_swapped(b, true);
}
// ... over a team of up to NT lanes; `turn` counts the calls.  Two buffers in turn: whoever writes one again has passed the barrier of the turn between, after which
// nobody still reads it.
template <int NT, typename F> __device__ __forceinline__ void team_sum2(F &a, F &b, int log, int turn, double2 (&lds)[2][NT / 64]) {
    lanes_sum2(a, b, log);
    if (log > 6) {
        double2 *p = lds[turn & 1];
        if ((threadIdx.x & 63) == 0) p[threadIdx.x >> 6] = double2{(double)a, (double)b};
        __syncthreads();
        const double2 wave = p[(threadIdx.x >> log << (log - 6)) + (threadIdx.x & ((1 << (log - 6)) - 1))];          // (a wave's lanes look at all of the team's)
        double s = wave.x, q = wave.y;
        lanes_sum2(s, q, log - 6);
        a = (F)s; b = (F)q;
    }
}

// ---- the pass back through the activation for one chunk of `valid` elements: xh and dy -> dz.  ReLU's gate: where 32 bits leave the sign of z open it is decided in
// 64, from the inputs in memory (x of the chunk at px, statistics and parameters of channel (c0 + e) % C): the gradient jumps there.  xh is off by at most 4 roundings.
template <int M> __device__ __forceinline__ void back_activation(const NormArgs &A, const T *px, int64_t n, int c0, int valid, const Mask<M> &mask, const float (&xh)[8], const float (&dy)[8],
                                                                             const float (&w)[8], const float (&b)[8], float (&dz)[8]) {
    if (A.act == PLENREG_ACT_RELU) {
        uint32_t open = 0, doubt = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float t = xh[e] * w[e], z = t + b[e];
            open |= z > 0.f ? 1u << e : 0u;
            doubt |= fabsf(z) <= 6e-7f * (fabsf(t) + fabsf(b[e])) ? 1u << e : 0u;
        }
        doubt &= (1u << valid) - 1u;
        const uint32_t kept_bits = doubt ? mask.bits() : 0u;
#pragma unroll 1
        while (doubt) {
            const int e = __ffs(doubt) - 1, c = (c0 + e) % A.C;
            doubt &= doubt - 1u;
            const double2 st = A.stats[n * A.G + c / A.D];
            const double v = kept_bits >> e & 1u ? (double)(float)px[e] : 0.0, wd = A.w ? (double)(float)((const W *)A.w)[c] : 1.0, bd = A.b ? (double)(float)((const W *)A.b)[c] : 0.0;
            open = (v - st.x) * st.y * wd + bd > 0.0 ? open | 1u << e : open & ~(1u << e);
        }
#pragma unroll
        for (int e = 0; e < 8; e++) dz[e] = open >> e & 1u ? dy[e] : 0.f;
    } else if (A.act == PLENREG_ACT_SILU) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float z = xh[e] * w[e] + b[e], s = logistic(z);
            dz[e] = dy[e] * (s * (1.f + z * (1.f - s)));
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) dz[e] = dy[e];
    }
}

// zeros behind the first `valid` elements of a partial chunk.  What stands there is another group's, and zero times its NaN or infinity would be none of the zeros that sums count on.
template <int V> __device__ __forceinline__ void clear_behind(float (&v)[8], int valid) {
    if (V) return;
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = e < valid ? v[e] : 0.f;
}

// ---- rows of one position (L = 1): a team of lanes per (row, group), K chunks per lane held in registers, one pass.  Teams of one wave join their sums by lane exchange,
//      wider ones through LDS.  A workgroup walks down the rows with its groups fixed, so that a lane keeps its channels: their parameters (and in the backward
//      pass their gradients) stay in registers.
struct RowPlace { int lane, gl, g, row; bool mine; };
template <int NT> __device__ __forceinline__ RowPlace row_place(const NormArgs &A, const RowPlan &P) {
    RowPlace p;
    const int team = threadIdx.x >> P.team_log;
    p.lane = threadIdx.x & ((1 << P.team_log) - 1);
    p.row = small_quotient(team, P.inv_gb);
    p.gl = team - p.row * P.gb;
    p.g = blockIdx.y * P.gb + p.gl;
    p.mine = p.row < P.rb && p.g < A.G;
    return p;
}
// first channel of chunk k of a lane within the row, and how much of the chunk belongs to the lane's group; lanes with nothing to do look at the last chunk of the last group
template <int K> __device__ __forceinline__ void row_chunks(const NormArgs &A, const RowPlan &P, const RowPlace &p, int (&c)[K], int (&valid)[K]) {
    const int g = p.g < A.G ? p.g : A.G - 1;
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int at = 8 * (p.lane + (k << P.team_log)), left = A.D - at;
        valid[k] = !p.mine || left < 0 ? 0 : left > 8 ? 8 : left;
        c[k] = g * A.D + (left > 0 ? at : (A.D - 1) & ~7);
    }
}
template <int V, bool STREAM> __device__ __forceinline__ void row_store(T *p, int valid, const float (&v)[8]) {
    if (V && STREAM) stream_store_whole<DT>(p, v);
    else if (V) store_whole<DT>(p, v);
    else store_chunk<DT>(p, valid, v);
}
// parameters of a lane's chunk, 1 / 0 where there are none
template <int V> __device__ __forceinline__ void row_params(const NormArgs &A, const void *p, int c0, float otherwise, float (&out)[8]) {
    if (p) {
        const Chunk<WT> c = load_inside<V, WT>((const W *)p, c0, A.C);
#pragma unroll
        for (int e = 0; e < 8; e++) out[e] = c.get(e);
        move_down<V>(out, c0, A.C);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) out[e] = otherwise;
    }
}

// Forward.  Bound by latency when small (100 x 512 f32: 2.8 us, a launch alone is 2.3), by vector issue when large: 16384 x 2048 bf16 with dropout and SiLU 34.6 us = 3.9 TB/s, 26
// instructions an element, of them 2.4 64-bit multiply-adds of the generator and 2 transcendentals at a quarter of the rate; its 134 MB alone would be 26 us.  4096 x 512 f32 6.2 us.
template <int V, int K, int NT, bool DROP, bool STREAM> __global__ __launch_bounds__(NT) void k_row_forward(NormArgs A, RowPlan P) {
    __shared__ double2 lds[2][NT / 64];
    const RowPlace p = row_place<NT>(A, P);
    int c[K], valid[K];
    row_chunks<K>(A, P, p, c, valid);
    // where a lane's row begins in x, in y and the mask (at), among the statistics: walked along by additions (a 64-bit product is a dozen slots); past the last row they stay
    const int64_t rows = (int64_t)gridDim.x * P.rb, x_step = rows * A.x_stride, step = rows * A.C, st_step = rows * A.G;
    int64_t n = (int64_t)blockIdx.x * P.rb + p.row, at = (n < A.N ? n : A.N - 1) * A.C, st_at = (n < A.N ? n : A.N - 1) * A.G + p.g;
    const T *px = (const T *)A.x + (n < A.N ? n : A.N - 1) * A.x_stride;
    Chunk<DT> x[K];
#pragma unroll
    for (int k = 0; k < K; k++) x[k] = load_inside<V, DT, STREAM>(px, c[k], A.C);
    float w[K][8], b[K][8];
#pragma unroll
    for (int k = 0; k < K; k++) { row_params<V>(A, A.w, c[k], 1.f, w[k]); row_params<V>(A, A.b, c[k], 0.f, b[k]); }
    Draw d = {};
    if (DROP) { d = make_draw(A.rng, A.site, A.cut); write_used(A); }
#pragma unroll 1
    for (int turn = 0; turn < P.trips; turn++) {
        const bool on = p.mine && n < A.N;
        const int64_t next = n + rows;
        const T *row = px;
        float v[K][8];
#pragma unroll
        for (int k = 0; k < K; k++) {
            const Mask<DROP ? V + 1 : 0> m(d, at + c[k]);
            unpack(x[k], v[k]);
            move_down<V>(v[k], c[k], A.C);
#pragma unroll
            for (int e = 0; e < 8; e++) v[k][e] = m.keep(e, v[k][e]);
        }
        if (turn + 1 < P.trips) {                               // the next row's, while this one is worked on
            if (next < A.N) px += x_step;
#pragma unroll
            for (int k = 0; k < K; k++) x[k] = load_inside<V, DT, STREAM>(px, c[k], A.C);
        }
        // s: the group's first element, after the mask
        float first;
        if (P.team_log <= 6) first = __shfl(v[0][0], (threadIdx.x & 63) >> P.team_log << P.team_log);
        else {
            first = (float)row[c[0] - 8 * p.lane];
            if (DROP && !kept(d, at + c[0] - 8 * p.lane)) first = 0.f;
        }
        const double shift = (double)first;
        double s = 0.0, q = 0.0;
#pragma unroll
        for (int k = 0; k < K; k++) {
            double sk = 0.0, qk = 0.0;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                if (!V && e >= valid[k]) v[k][e] = first;                                    // what is not there adds nothing
                const double t = (double)v[k][e] - shift;
                sk += t; qk = fma(t, t, qk);
            }
            s += !V || valid[k] ? sk : 0.0; q += !V || valid[k] ? qk : 0.0;
        }
        team_sum2<NT>(s, q, P.team_log, turn, lds);
        const double2 st = finish_stats(A, A.count, shift, s, q);
        if (on) {
            if (A.stats && p.lane == 0) A.stats[st_at] = st;
            const float mean = (float)st.x, rstd = (float)st.y, offset = -(float)(st.x - (double)mean) * rstd;
#pragma unroll
            for (int k = 0; k < K; k++) {
                if (!valid[k]) continue;
#pragma unroll
                for (int e = 0; e < 8; e++) v[k][e] = from_mean(v[k][e], mean, rstd, offset) * w[k][e] + b[k][e];
                activate(v[k], A.act);
                row_store<V, STREAM>((T *)A.out + at + c[k], valid[k], v[k]);
            }
        }
        n = next;
        if (n < A.N) { at += step; st_at += st_step; }
    }
}

// Backward of the rows: one chunk a lane where that is enough, since x, dy, dz, two parameters and their two gradients are held per element (two chunks: 200 registers, half the waves).  Sums
// of a row in 32 bits: at most 8192 elements in a tree.  16384 x 2048 bf16 with dropout and SiLU 50 us, vector issue (44 instructions an element; its 201 MB alone would be 39 us); 4096 x 512
// f32 10 us, 100 x 512 6 us; 8192 x 8192 bf16 117 us (as two launches that read x and dy again 174).  Each workgroup leaves one row of partial parameter gradients: part[blockIdx.x][0 / 1][C] = dw, db of its rows, summed over its teams in LDS.
template <int V, int K, int NT, bool DROP, bool STREAM> __global__ __launch_bounds__(NT) void k_row_backward(NormArgs A, RowPlan P, float *part) {
    __shared__ double2 lds[2][NT / 64];
    __shared__ float joined[NT * 8 * K];
    const RowPlace p = row_place<NT>(A, P);
    int c[K], valid[K];
    row_chunks<K>(A, P, p, c, valid);
    const int g0 = p.g < A.G ? p.g : A.G - 1;
    // (as in the forward pass, additions instead of products)
    const int64_t rows = (int64_t)gridDim.x * P.rb, x_step = rows * A.x_stride, dy_step = rows * A.dy_stride, step = rows * A.C, st_step = rows * A.G;
    int64_t n = (int64_t)blockIdx.x * P.rb + p.row, at = (n < A.N ? n : A.N - 1) * A.C;
    const T *px = (const T *)A.x + (n < A.N ? n : A.N - 1) * A.x_stride, *pdy = (const T *)A.dy + (n < A.N ? n : A.N - 1) * A.dy_stride;
    const double2 *pst = A.stats + (n < A.N ? n : A.N - 1) * A.G + g0;
    Chunk<DT> x[K], g[K];
#pragma unroll
    for (int k = 0; k < K; k++) { x[k] = load_inside<V, DT, STREAM>(px, c[k], A.C); g[k] = load_inside<V, DT, STREAM>(pdy, c[k], A.C); }
    double2 st = *pst;
    float w[K][8], b[K][8], dw[K][8] = {}, db[K][8] = {};
#pragma unroll
    for (int k = 0; k < K; k++) { row_params<V>(A, A.w, c[k], 1.f, w[k]); row_params<V>(A, A.b, c[k], 0.f, b[k]); clear_behind<V>(w[k], valid[k]); }
    Draw d = {};
    if (DROP) d = make_draw(A.rng, A.site, A.cut);
#pragma unroll 1
    for (int turn = 0; turn < P.trips; turn++) {
        const bool on = n < A.N && valid[0];
        float xh[K][8] = {}, gw[K][8] = {}, s = 0.f, q = 0.f, rstd = 0.f;
        Mask<DROP ? V + 1 : 0> m[K];
#pragma unroll
        for (int k = 0; k < K; k++) {
            m[k] = Mask<DROP ? V + 1 : 0>(d, at + c[k]);
            if (on && (K == 1 || valid[k])) {
                const float mean = (float)st.x, rest = (float)(st.x - (double)mean);
                rstd = (float)st.y;
                float dy[8], dz[8];
                unpack(x[k], xh[k]);
                unpack(g[k], dy);
                move_down<V>(xh[k], c[k], A.C);
                move_down<V>(dy, c[k], A.C);
#pragma unroll
                for (int e = 0; e < 8; e++) xh[k][e] = ((m[k].keep(e, xh[k][e]) - mean) - rest) * rstd;
                clear_behind<V>(xh[k], valid[k]);
                back_activation(A, px + c[k], n, c[k], valid[k], m[k], xh[k], dy, w[k], b[k], dz);
                clear_behind<V>(dz, valid[k]);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    gw[k][e] = dz[e] * w[k][e];
                    s += gw[k][e]; q = fmaf(gw[k][e], xh[k][e], q);
                    db[k][e] += dz[e]; dw[k][e] = fmaf(dz[e], xh[k][e], dw[k][e]);
                }
            }
        }
        const int64_t here = at;
        n += rows;
        if (n < A.N) { px += x_step; pdy += dy_step; pst += st_step; at += step; }
        if (turn + 1 < P.trips) {                               // the next row's, while this one's sums are joined
#pragma unroll
            for (int k = 0; k < K; k++) { x[k] = load_inside<V, DT, STREAM>(px, c[k], A.C); g[k] = load_inside<V, DT, STREAM>(pdy, c[k], A.C); }
            st = *pst;
        }
        team_sum2<NT>(s, q, P.team_log, turn, lds);
        if (on) {
            const float m1 = s * (float)A.inv_count, m2 = q * (float)A.inv_count;
#pragma unroll
            for (int k = 0; k < K; k++) {
                if (K > 1 && !valid[k]) continue;
#pragma unroll
                for (int e = 0; e < 8; e++) gw[k][e] = m[k].keep(e, rstd * (gw[k][e] - m1 - xh[k][e] * m2));
                row_store<V, STREAM>((T *)A.out + here + c[k], valid[k], gw[k]);
            }
        }
    }
    if (!part) return;
    const int width = 8 * K << P.team_log, columns = P.gb * width;              // joined[row][group of the workgroup][channel of the group, padded to whole chunks]
#pragma unroll 1
    for (int pass = 0; pass < 2; pass++) {
        __syncthreads();
        if (p.row < P.rb)
#pragma unroll
            for (int k = 0; k < K; k++)
#pragma unroll
                for (int e = 0; e < 8; e++) joined[p.row * columns + p.gl * width + 8 * (p.lane + (k << P.team_log)) + e] = pass ? db[k][e] : dw[k][e];
        __syncthreads();
        for (int j = threadIdx.x; j < columns; j += NT) {
            const int gj = j >> (P.team_log + 2 + K), cc = j & (width - 1), gg = blockIdx.y * P.gb + gj;
            if (gg >= A.G || cc >= A.D) continue;
            float t = 0.f;
            for (int r = 0; r < P.rb; r++) t += joined[r * columns + j];
            part[((int64_t)blockIdx.x * 2 + pass) * A.C + gg * A.D + cc] = t;
        }
    }
}

// dw, db = column sums of part[rows][2][C] in 64 bits (a fixed order instead of atomics; 3.4 us for 512 rows of 2 x 512, mostly launch, 4.3 for 2 x 2048): 16 columns per workgroup, blockDim / 16 rows at a time.  lds: [blockDim / 16][17]
__device__ __forceinline__ void param_columns(const NormArgs &A, const float *part, int rows, int block, void *dw, void *db, double *lds) {
    const int64_t width = 2 * (int64_t)A.C, column = (int64_t)block * 16 + (threadIdx.x & 15);
    const int r0 = threadIdx.x >> 4, step = blockDim.x >> 4;
    double s = 0.0;
    if (column < width) {
        int r = r0;
        for (; r + 7 * step < rows; r += 8 * step) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = part[(r + k * step) * width + column];
#pragma unroll
            for (int k = 0; k < 8; k++) s += (double)v[k];
        }
        for (; r < rows; r += step) s += (double)part[r * width + column];
    }
    lds[r0 * 17 + (threadIdx.x & 15)] = s;
    __syncthreads();
    if (threadIdx.x < 256) {
        // column t / 16, rows t % 16 + 16 k: then over 16 lanes
        const int col = threadIdx.x >> 4;
        double t = 0.0, unused = 0.0;
        for (int r = threadIdx.x & 15; r < step; r += 16) t += lds[r * 17 + col];
        lanes_sum2(t, unused, 4);
        const int64_t c = (int64_t)block * 16 + col;
        if ((threadIdx.x & 15) == 0 && c < width) {
            void *to = c < A.C ? dw : db;
            if (to) ((W *)to)[c < A.C ? c : c - A.C] = (W)(float)t;
        }
    }
}
__global__ __launch_bounds__(1024) void k_row_params(NormArgs A, const float *part, int rows, void *dw, void *db) {
    __shared__ double lds[64 * 17];
    param_columns(A, part, rows, blockIdx.x, dw, db, lds);
}

// ---- rows too wide for a workgroup's registers: one workgroup goes over a group twice, the second time out of the caches; the parameters are read with each chunk.  Its parameter gradients
//      are a launch of their own, in which a thread owns a chunk column and walks down the rows.  4096 x 16384 bf16: forward 62 us = 4.3 TB/s, backward 177 (memory: x and dy come from
//      there twice, once for either launch); as slabs of one position 198 and 628.
template <int V> __device__ __forceinline__ int wide_valid(const NormArgs &A, int off) { return V || A.D - off > 8 ? 8 : A.D - off; }
// forward; grid: (n, g) pairs
template <int V, bool DROP, bool STREAM> __global__ __launch_bounds__(WIDE_NT) void k_wide_forward(NormArgs A) {
    __shared__ double2 lds[2][WIDE_NT / 64];
    Draw d = {};
    if (DROP) { d = make_draw(A.rng, A.site, A.cut); write_used(A); }
    int turn = 0;
#pragma unroll 1
    for (int64_t item = blockIdx.x; item < A.N * A.G; item += gridDim.x, turn++) {
        const int64_t n = item / A.G;
        const int c0 = (int)(item - n * A.G) * A.D;
        const T *px = (const T *)A.x + n * A.x_stride;
        float first = (float)px[c0];
        if (DROP && !kept(d, n * A.C + c0)) first = 0.f;
        const double shift = (double)first;
        double s = 0.0, q = 0.0;
        int off = 8 * threadIdx.x;
        Chunk<DT> x = load_inside<V, DT>(px, c0 + (off < A.D ? off : 0), A.C);
#pragma unroll 1
        for (; off < A.D; off += 8 * WIDE_NT) {
            float v[8];
            unpack(x, v);
            move_down<V>(v, c0 + off, A.C);
            const int next = off + 8 * WIDE_NT, valid = wide_valid<V>(A, off);
            x = load_inside<V, DT>(px, c0 + (next < A.D ? next : off), A.C);
            const Mask<DROP ? V + 1 : 0> m(d, n * A.C + c0 + off);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const double t = !V && e >= valid ? 0.0 : (double)m.keep(e, v[e]) - shift;
                s += t; q = fma(t, t, q);
            }
        }
        team_sum2<WIDE_NT>(s, q, WIDE_LOG, turn, lds);
        const double2 st = finish_stats(A, A.count, shift, s, q);
        if (A.stats && threadIdx.x == 0) A.stats[item] = st;
        const float mean = (float)st.x, rstd = (float)st.y, offset = -(float)(st.x - (double)mean) * rstd;
        T *y = (T *)A.out + n * A.C + c0;
        off = 8 * threadIdx.x;
        x = load_inside<V, DT, STREAM>(px, c0 + (off < A.D ? off : 0), A.C);
#pragma unroll 1
        for (; off < A.D; off += 8 * WIDE_NT) {
            float v[8], w[8], b[8];
            unpack(x, v);
            move_down<V>(v, c0 + off, A.C);
            const int next = off + 8 * WIDE_NT;
            x = load_inside<V, DT, STREAM>(px, c0 + (next < A.D ? next : off), A.C);
            row_params<V>(A, A.w, c0 + off, 1.f, w);
            row_params<V>(A, A.b, c0 + off, 0.f, b);
            const Mask<DROP ? V + 1 : 0> m(d, n * A.C + c0 + off);
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = from_mean(m.keep(e, v[e]), mean, rstd, offset) * w[e] + b[e];
            activate(v, A.act);
            row_store<V, STREAM>(y + off, wide_valid<V>(A, off), v);
        }
    }
}
// dz, xh and w of a chunk (zeros behind the group's end)
template <int V, bool DROP>
__device__ __forceinline__ void wide_back(const NormArgs &A, const Mask<DROP ? V + 1 : 0> &m, const Chunk<DT> &x, const Chunk<DT> &g, const T *px, int64_t n, int c, int valid, double2 st, float (&w)[8], float (&xh)[8],
                                          float (&dz)[8]) {
    float b[8], dy[8];
    row_params<V>(A, A.w, c, 1.f, w);
    row_params<V>(A, A.b, c, 0.f, b);
    unpack(x, xh);
    unpack(g, dy);
    move_down<V>(xh, c, A.C);
    move_down<V>(dy, c, A.C);
    const float mean = (float)st.x, rest = (float)(st.x - (double)mean), rstd = (float)st.y;
#pragma unroll
    for (int e = 0; e < 8; e++) xh[e] = ((m.keep(e, xh[e]) - mean) - rest) * rstd;
    clear_behind<V>(xh, valid);
    clear_behind<V>(w, valid);
    back_activation(A, px + c, n, c, valid, m, xh, dy, w, b, dz);
    clear_behind<V>(dz, valid);
}
// the gradient of x; grid: (n, g) pairs.  (Sums in 32 bits: a lane adds at most 64 elements before the lanes are joined.)
template <int V, bool DROP, bool STREAM> __global__ __launch_bounds__(WIDE_NT) void k_wide_backward(NormArgs A) {
    __shared__ double2 lds[2][WIDE_NT / 64];
    Draw d = {};
    if (DROP) d = make_draw(A.rng, A.site, A.cut);
    int turn = 0;
#pragma unroll 1
    for (int64_t item = blockIdx.x; item < A.N * A.G; item += gridDim.x, turn++) {
        const int64_t n = item / A.G;
        const int c0 = (int)(item - n * A.G) * A.D;
        const T *px = (const T *)A.x + n * A.x_stride, *pdy = (const T *)A.dy + n * A.dy_stride;
        const double2 st = A.stats[item];
        float s = 0.f, q = 0.f, xh[8], dz[8], w[8];
        int off = 8 * threadIdx.x;
        Chunk<DT> x = load_inside<V, DT>(px, c0 + (off < A.D ? off : 0), A.C), g = load_inside<V, DT>(pdy, c0 + (off < A.D ? off : 0), A.C);
#pragma unroll 1
        for (; off < A.D; off += 8 * WIDE_NT) {
            const Chunk<DT> xn = x, gn = g;
            const int next = off + 8 * WIDE_NT, at = c0 + (next < A.D ? next : off);
            x = load_inside<V, DT>(px, at, A.C); g = load_inside<V, DT>(pdy, at, A.C);
            const Mask<DROP ? V + 1 : 0> m(d, n * A.C + c0 + off);
            wide_back<V, DROP>(A, m, xn, gn, px, n, c0 + off, wide_valid<V>(A, off), st, w, xh, dz);
#pragma unroll
            for (int e = 0; e < 8; e++) { const float gw = dz[e] * w[e]; s += gw; q = fmaf(gw, xh[e], q); }
        }
        team_sum2<WIDE_NT>(s, q, WIDE_LOG, turn, lds);
        const float m1 = s * (float)A.inv_count, m2 = q * (float)A.inv_count, rstd = (float)st.y;
        T *dx = (T *)A.out + n * A.C + c0;
        off = 8 * threadIdx.x;
        x = load_inside<V, DT, STREAM>(px, c0 + (off < A.D ? off : 0), A.C); g = load_inside<V, DT, STREAM>(pdy, c0 + (off < A.D ? off : 0), A.C);
#pragma unroll 1
        for (; off < A.D; off += 8 * WIDE_NT) {
            const Chunk<DT> xn = x, gn = g;
            const int next = off + 8 * WIDE_NT, at = c0 + (next < A.D ? next : off), valid = wide_valid<V>(A, off);
            x = load_inside<V, DT, STREAM>(px, at, A.C); g = load_inside<V, DT, STREAM>(pdy, at, A.C);
            const Mask<DROP ? V + 1 : 0> m(d, n * A.C + c0 + off);
            wide_back<V, DROP>(A, m, xn, gn, px, n, c0 + off, valid, st, w, xh, dz);
#pragma unroll
            for (int e = 0; e < 8; e++) dz[e] = m.keep(e, rstd * (dz[e] * w[e] - m1 - xh[e] * m2));
            row_store<V, STREAM>(dx + off, valid, dz);
        }
    }
}
// part[split][0 / 1][C] = dw, db of rows split, split + splits, ...; grid: blocks of 256 chunk columns (per group: its chunks), splits
template <int V, bool DROP> __global__ __launch_bounds__(256) void k_wide_params(NormArgs A, float *part) {
    const int per = (A.D + 7) >> 3, j = blockIdx.x * 256 + threadIdx.x;
    if (j >= per * A.G) return;
    const int grp = j / per, off = 8 * (j - grp * per), c = grp * A.D + off, valid = wide_valid<V>(A, off);
    Draw d = {};
    if (DROP) d = make_draw(A.rng, A.site, A.cut);
    int64_t n = blockIdx.y;
    const T *px = (const T *)A.x + n * A.x_stride, *pdy = (const T *)A.dy + n * A.dy_stride;
    Chunk<DT> x = load_inside<V, DT>(px, c, A.C), g = load_inside<V, DT>(pdy, c, A.C);
    double2 st = A.stats[n * A.G + grp];
    float dw[8] = {}, db[8] = {};
#pragma unroll 1
    for (; n < A.N; n += gridDim.y) {
        const Chunk<DT> xn = x, gn = g;
        const double2 now = st;
        const T *here = px;
        if (n + gridDim.y < A.N) { px += gridDim.y * A.x_stride; pdy += gridDim.y * A.dy_stride; st = A.stats[(n + gridDim.y) * A.G + grp]; }
        x = load_inside<V, DT>(px, c, A.C); g = load_inside<V, DT>(pdy, c, A.C);
        const Mask<DROP ? V + 1 : 0> m(d, n * A.C + c);
        float w[8], xh[8], dz[8];
        wide_back<V, DROP>(A, m, xn, gn, here, n, c, valid, now, w, xh, dz);
#pragma unroll
        for (int e = 0; e < 8; e++) { db[e] += dz[e]; dw[e] = fmaf(dz[e], xh[e], dw[e]); }
    }
    float *to = part + (int64_t)blockIdx.y * 2 * A.C + c;
#pragma unroll
    for (int e = 0; e < 8; e++)
        if (e < valid) { to[e] = dw[e]; to[A.C + e] = db[e]; }
}

// ---- many positions: a slab is size = L C contiguous elements, seen as rows of q C (q = the smallest number of positions that
//      fill whole chunks, so that odd channel counts load whole chunks too; the last row may be cut short, and of its last chunk there may be a part).  A thread owns one
//      chunk column (8 fixed virtual channels v, channel v % C) and walks down the rows; workgroups split the rows and, where they are wide, the columns.  Statistics, their
//      join, and the result are launches of their own: the second reading of x comes out of the caches while it fits.
struct Column { int first, col, r; bool mine; };
__device__ __forceinline__ Column my_column(const MapPlan &P, int col_block) {
    Column c;
    c.first = col_block * P.bcol;
    c.r = small_quotient(threadIdx.x, P.inv_bcol);
    c.col = c.first + (int)threadIdx.x - c.r * P.bcol;
    c.mine = c.r < P.R && c.col < P.ncol;
    if (c.col >= P.ncol) c.col = P.ncol - 1;             // (of the last, narrower block: its idle threads look at the parameters of the last column, not behind them)
    return c;
}
// a workgroup's rows of slab n: `base` elements into it, `lim` elements; a thread takes the chunks at off, off + step, ... that are whole, and if it then stands at off < lim,
// the slab's last, partial chunk.  (Spans are below 2^28 elements: offsets in 32 bits, what is the same for the workgroup in scalar registers.)
struct Span { int64_t base; int lim, off, step; };
__device__ __forceinline__ Span my_span(const NormArgs &A, const MapPlan &P, const Column &c, int64_t rows_per) {
    Span t;
    const int width = A.C << P.q_log;
    t.base = blockIdx.x * rows_per * width;
    const int64_t left = A.size - t.base;
    t.lim = left < rows_per * width ? (int)left : (int)(rows_per * width);
    t.step = P.R * width;
    t.off = c.r * width + 8 * c.col;
    return t;
}
// the chunk at off, or the span's last whole one (a load under a condition would wait for the ones before it); lim >= 8.  STREAM: past the caches
template <bool STREAM = false> __device__ __forceinline__ Chunk<DT> span_load(const T *p, const Span &t, int off) {
    p += off < t.lim - 8 ? off : t.lim - 8;
    return STREAM ? stream_whole<DT>(p) : load_whole<DT>(p);
}

// channel and group of the first of a thread's virtual channels; `next` steps to the one after
struct Channel {
    int c, g, d;
    __device__ __forceinline__ Channel(const NormArgs &A, int v) {
        c = v - small_quotient(v, A.inv_C) * A.C;
        g = small_quotient(c, A.inv_D);
        d = c - g * A.D;
    }
    __device__ __forceinline__ void next(const NormArgs &A) {
        c++; d++;
        if (d == A.D) { d = 0; g++; }
        if (c == A.C) { c = 0; g = 0; }
    }
};
struct Nothing { __device__ __forceinline__ float operator()(int) const { return 0.f; } };
// sums over the workgroup's threads of a[8], b[8] per virtual channel, joined per group: result(g, before(g), sums) from one lane each (zeros for a group with no channel in this
// workgroup's columns); before: what the result has to wait for, asked for first.
// A thread leaves one pair per group that its chunk can reach: one (V = 2), two (groups of 8 and more channels) or eight.  `lds`: blockDim.x times as many.
// (8 x 4096 x 320 with 32 groups, forward sums: 9.1 us with eight pairs always and the copies of a row one after the other; without any join 5.4.)
template <int V, class B, class F>
__device__ __forceinline__ void join_groups(const double (&a)[8], const double (&b)[8], const NormArgs &A, const MapPlan &P, const Column &c, double2 *lds, B before, F result) {
    const int NT = blockDim.x;
    int at = c.r * P.bcol + c.col - c.first;
    asm volatile("" : "+v"(at));                     // (hidden, as the column in load_constants: in a loop over slabs the addresses would be kept)
    const bool two = V == 1 && A.D >= 8;
    __syncthreads();
    if (c.mine) {
        if (V == 2) lds[at] = double2{((a[0] + a[1]) + (a[2] + a[3])) + ((a[4] + a[5]) + (a[6] + a[7])), ((b[0] + b[1]) + (b[2] + b[3])) + ((b[4] + b[5]) + (b[6] + b[7]))};
        else if (two) {
            const int split = A.D - Channel(A, 8 * c.col).d;
            double a0 = 0.0, a1 = 0.0, b0 = 0.0, b1 = 0.0;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                a0 += e < split ? a[e] : 0.0; b0 += e < split ? b[e] : 0.0;
                a1 += e < split ? 0.0 : a[e]; b1 += e < split ? 0.0 : b[e];
            }
            lds[at] = double2{a0, b0};
            lds[NT + at] = double2{a1, b1};
        } else
#pragma unroll
            for (int e = 0; e < 8; e++) lds[e * NT + at] = double2{a[e], b[e]};
    }
    __syncthreads();
    // a group's entries: copy k of the row, row r, and u: its chunks, or (groups of less than 8 channels) its channels
    int thread = threadIdx.x;
    asm volatile("" : "+v"(thread));
    const int lane = thread & ((1 << P.lanes_log) - 1), teams = NT >> P.lanes_log, units = V == 2 ? A.D >> 3 : two ? (A.D + 14) >> 3 : A.D, entries = units * P.R << P.q_log;
    const int end = c.first + P.bcol < P.ncol ? c.first + P.bcol : P.ncol;
    const float inv_units = 1.f / (float)units, inv_R = 1.f / (float)P.R;
#pragma unroll 1
    for (int g0 = 0; g0 < A.G; g0 += teams) {                        // (every lane takes every turn: the exchange needs them all)
        const int g = g0 + (thread >> P.lanes_log);
        const float first = before(g < A.G ? g : A.G - 1);
        double s = 0.0, q = 0.0;
        if (g < A.G)
#pragma unroll 1
            for (int i = lane; i < entries; i += 1 << P.lanes_log) {
                const int kr = small_quotient(i, inv_units), u = i - kr * units, k = small_quotient(kr, inv_R), r = kr - k * P.R;
                const int lo = k * A.C + g * A.D, col = V == 2 || two ? (lo >> 3) + u : (lo + u) >> 3;
                if (col < c.first || col >= end || (two && 8 * col >= lo + A.D)) continue;
                const double2 t = lds[(V == 2 ? 0 : two ? (8 * col < lo ? NT : 0) : ((lo + u) & 7) * NT) + r * P.bcol + col - c.first];
                s += t.x; q += t.y;
            }
        lanes_sum2(s, q, P.lanes_log);
        if (g < A.G && lane == 0) result(g, first, s, q);
    }
}
// sums over the `splits` partial pairs of one (n, g), by one wave
__device__ __forceinline__ double2 join_splits(const double2 *part, int splits) {
    double s = 0.0, q = 0.0;
    for (int k = threadIdx.x & 63; k < splits; k += 64) { const double2 t = part[k]; s += t.x; q += t.y; }
    lanes_sum2(s, q, 6);
    return double2{s, q};
}
// the sums over the partial pairs of every group of a slab, by a whole workgroup: before and result as in join_groups
template <class B, class F> __device__ __forceinline__ void join_slab(const NormArgs &A, const MapPlan &P, const double2 *part, B before, F result) {
    const int parts = P.splits * P.col_blocks, step = 1 << P.join_log, lane = threadIdx.x & (step - 1), teams = blockDim.x >> P.join_log;
#pragma unroll 1
    for (int g0 = 0; g0 < A.G; g0 += teams) {                        // (every lane takes every turn: the exchange needs them all)
        const int g = g0 + (threadIdx.x >> P.join_log);
        const double2 *p = part + (int64_t)(g < A.G ? g : A.G - 1) * parts;
        const float first = before(g < A.G ? g : A.G - 1);
        double s = 0.0, q = 0.0;
#pragma unroll 1
        for (int k = lane; k < parts; k += 8 * step) {
            double2 t[8];
#pragma unroll
            for (int j = 0; j < 8; j++) t[j] = p[k + j * step < parts ? k + j * step : k];
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (k + j * step < parts) { s += t[j].x; q += t[j].y; }
        }
        lanes_sum2(s, q, P.join_log);
        if (g < A.G && lane == 0) result(g, first, s, q);
    }
}
// s of a group of a slab: its first element, after the mask.  (Not one for all of them: groups far from it would lose their variance, and its NaN or infinity would be theirs.)
template <bool DROP> __device__ __forceinline__ float group_shift(const NormArgs &A, const Draw &d, int64_t n, int g) {
    const float v = (float)((const T *)A.x)[n * A.x_stride + g * A.D];
    return DROP && !kept(d, n * A.size + g * A.D) ? 0.f : v;
}
// ... of a thread's 8 virtual channels (V = 2: one group, element 0).  Masked and of more than two groups to a chunk: drawn once per group and shared in `lds` (G floats of the join's space),
// rather than up to eight times by every thread.
template <int V, bool DROP> __device__ __forceinline__ void load_shifts(const NormArgs &A, const Draw &d, int col, int64_t n, double2 *lds, float (&s)[V == 2 ? 1 : 8]) {
    asm volatile("" : "+v"(col));                    // (as in load_constants)
    Channel ch(A, 8 * col);
    if (V == 2) s[0] = group_shift<DROP>(A, d, n, ch.g);
    else if (A.D >= 8) {                             // the chunk reaches into one more group at most
        const int split = A.D - ch.d;
        const float s0 = group_shift<DROP>(A, d, n, ch.g), s1 = group_shift<DROP>(A, d, n, ch.g + 1 < A.G ? ch.g + 1 : 0);
#pragma unroll
        for (int e = 0; e < (V == 2 ? 1 : 8); e++) s[e] = e < split ? s0 : s1;
    } else {
        float *all = (float *)lds;
        if (DROP) {
            __syncthreads();
            int g = threadIdx.x;
            asm volatile("" : "+v"(g));
            for (; g < A.G; g += blockDim.x) all[g] = group_shift<DROP>(A, d, n, g);
            __syncthreads();
        }
#pragma unroll
        for (int e = 0; e < (V == 2 ? 1 : 8); e++) { s[e] = DROP ? all[ch.g] : group_shift<DROP>(A, d, n, ch.g); ch.next(A); }
    }
}

// s, q += the sums of (x - s), (x - s)^2 of a span of slab n, per virtual channel.  LEAN: a chunk's eight shifts stay in 32 bits until their use; carried in 64 bits through the loop they cost
// one or two waves a SIMD, converted at each use 8 instructions a chunk.  Split sums with more than two workgroups a compute unit, 1024 x 512 x 320: both forward launches 199 -> 176 us; slabs of one
// workgroup with dropout, 20000 x 16 x 66: 371 -> 332.  Where fewer waves are there it loses: split sums of 8 x 4096 x 320 8.1 -> 8.6, slabs 8 x 32 x 320 without dropout 6.9 -> 7.1.
template <int V, bool DROP, bool LEAN> __device__ __forceinline__ void span_sums(const NormArgs &A, const Draw &d, const Column &c, const Span &t, int64_t n, double2 *lds, double (&s)[8], double (&q)[8]) {
    const T *x = (const T *)A.x + n * A.x_stride + t.base;
    int off = t.off;
    Chunk<DT> v;
    if (t.lim >= 8) v = span_load(x, t, off);
    float shift[V == 2 ? 1 : 8];
    load_shifts<V, DROP>(A, d, c.col, n, lds, shift);
    const auto add = [&](const Chunk<DT> &chunk, int valid) {
        float f[8];
        unpack(chunk, Mask<DROP ? V : 0>(d, n * A.size + t.base + off), f);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            if (V == 1 && LEAN) asm("" : "+v"(shift[V == 2 ? 0 : e]));
            const double u = e < valid ? (double)f[e] - (double)shift[V == 2 ? 0 : e] : 0.0;
            s[e] += u; q[e] = fma(u, u, q[e]);
        }
    };
    if (!c.mine) return;
#pragma unroll 1
    while (off + 8 <= t.lim) {
        const Chunk<DT> now = v;
        v = span_load(x, t, off + t.step);             // the next chunk is on its way while this one is added
        add(now, 8);
        off += t.step;
    }
    if (V == 1 && off < t.lim) add(load_chunk<DT>(x + off, t.lim - off), t.lim - off);
}
// part[n][g][split][column block] = sums of (x - s), (x - s)^2.  Grid: splits, column blocks, slabs.  2 x 262144 x 128 bf16 26 us = 5.2 TB/s (memory; a kernel that only reads gets to 6.3);
// 8 x 4096 x 320 8.2 us, latency: 5.4 for the reading by 2.5 waves a SIMD, the rest the groups' shifts (0.3) and the join.  (Two or three chunks on their way instead of one: no faster.)
template <int V, bool DROP, bool LEAN> __global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(DROP || !LEAN ? 5 : 6, 8))) void k_map_sums(NormArgs A, MapPlan P, double2 *part) {
    extern __shared__ double2 lds[];
    const Column c = my_column(P, blockIdx.y);
    const Span t = my_span(A, P, c, P.rows_per);
    Draw d = {};
    if (DROP) { d = make_draw(A.rng, A.site, A.cut); write_used(A); }
#pragma unroll 1
    for (int64_t n = blockIdx.z; n < A.N; n += gridDim.z) {
        double s[8] = {}, q[8] = {};
        span_sums<V, DROP, LEAN>(A, d, c, t, n, lds, s, q);
        const int64_t parts = (int64_t)P.splits * P.col_blocks;
        double2 *out = part + n * A.G * parts + blockIdx.x * P.col_blocks + blockIdx.y;
        join_groups<V>(s, q, A, P, c, lds, Nothing(), [&](int g, float, double a, double b) { out[g * parts] = double2{a, b}; });
    }
}
// one wave per (n, g), where a slab has too many partial pairs for every workgroup of the result to join them: ~4.3 us, a launch and two dependent loads
template <bool DROP> __global__ __launch_bounds__(256) void k_map_stats(NormArgs A, int splits, const double2 *part) {
    Draw d = {};
    if (DROP) d = make_draw(A.rng, A.site, A.cut);
    for (int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); item < A.N * A.G; item += (int64_t)gridDim.x * 4) {
        const int64_t n = item / A.G;
        const double shift = group_shift<DROP>(A, d, n, (int)(item - n * A.G));
        const double2 t = join_splits(part + item * splits, splits);
        if ((threadIdx.x & 63) == 0) A.stats[item] = finish_stats(A, A.count, shift, t.x, t.y);
    }
}
// statistics and parameters of a thread's 8 virtual channels (V = 2: one group, statistics in element 0).
// (The column is hidden from the compiler: it would keep every address of a loop over slabs in registers, and spill.)
template <int V> struct Constants { float mean[V == 2 ? 1 : 8], rest[V == 2 ? 1 : 8], rstd[V == 2 ? 1 : 8], w[8], b[8]; };
template <int V> __device__ __forceinline__ void load_constants(const NormArgs &A, const MapPlan &P, const double2 *stats, int col, Constants<V> &k) {
    asm volatile("" : "+v"(col));
    Channel ch(A, 8 * col);
    if (P.q_log == 0) {                         // (columns do not wrap: the parameters as whole chunks)
        row_params<1>(A, A.w, 8 * col, 1.f, k.w);
        row_params<1>(A, A.b, 8 * col, 0.f, k.b);
    } else {
        // (all loads of one kind under one condition: each would wait for the one before)
#pragma unroll
        for (int e = 0; e < 8; e++) { k.w[e] = 1.f; k.b[e] = 0.f; }
        const auto gather = [&](const void *p, float (&out)[8]) {
            int at = ch.c;
#pragma unroll
            for (int e = 0; e < 8; e++) { out[e] = (float)((const W *)p)[at]; at = at + 1 < A.C ? at + 1 : 0; }
        };
        if (A.w) gather(A.w, k.w);
        if (A.b) gather(A.b, k.b);
    }
    const double2 st = stats[ch.g];
    const float mean = (float)st.x, rest = (float)(st.x - (double)mean), rstd = (float)st.y;
    if (V == 2) { k.mean[0] = mean; k.rest[0] = rest; k.rstd[0] = rstd; return; }
    if (A.D >= 8) {                                         // the chunk reaches into one more group at most
        const int split = A.D - ch.d;
        const double2 st1 = stats[ch.g + 1 < A.G ? ch.g + 1 : 0];
        const float mean1 = (float)st1.x, rest1 = (float)(st1.x - (double)mean1), rstd1 = (float)st1.y;
#pragma unroll
        for (int i = 0; i < (V == 2 ? 1 : 8); i++) { k.mean[i] = i < split ? mean : mean1; k.rest[i] = i < split ? rest : rest1; k.rstd[i] = i < split ? rstd : rstd1; }
    } else
#pragma unroll
        for (int i = 0; i < (V == 2 ? 1 : 8); i++) {
            const double2 t = stats[ch.g];
            k.mean[i] = (float)t.x; k.rest[i] = (float)(t.x - (double)k.mean[i]); k.rstd[i] = (float)t.y;
            ch.next(A);
        }
}
template <int V> __device__ __forceinline__ void normalise(const Constants<V> &k, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; e++) { const int i = V == 2 ? 0 : e; v[e] = ((v[e] - k.mean[i]) - k.rest[i]) * k.rstd[i]; }
}
// the results of a span of slab n; ready() -> the slab's statistics
template <int V, bool DROP, bool STREAM, class F> __device__ __forceinline__ void span_apply(const NormArgs &A, const MapPlan &P, const Draw &d, const Column &c, const Span &t, int64_t n, F ready) {
    const T *x = (const T *)A.x + n * A.x_stride + t.base;
    T *y = (T *)A.out + n * A.size + t.base;
    int off = t.off;
    Chunk<DT> v;
    if (t.lim >= 8) v = span_load<STREAM>(x, t, off);
    Constants<V> k;
    load_constants<V>(A, P, ready(), c.col, k);
#pragma unroll
    for (int e = 0; e < 8; e++) {
        // the result is (x - mean) w' + b', w' = w rstd, b' = b - rest w' (of an infinite w' the largest, so that no 0 inf comes in).  The mean's second word subtracted from each element instead: 1024 x 512 x 320 179 -> 214 us, registers.
        const int i = V == 2 ? 0 : e;
        k.w[e] *= k.rstd[i];
        k.b[e] = fmaf(-k.rest[i], __builtin_amdgcn_fmed3f(k.w[e], -3e38f, 3e38f), k.b[e]);
    }
    const auto result = [&](const Chunk<DT> &chunk, float (&f)[8]) {
        unpack(chunk, Mask<DROP ? V : 0>(d, n * A.size + t.base + off), f);
#pragma unroll
        for (int e = 0; e < 8; e++) f[e] = (f[e] - k.mean[V == 2 ? 0 : e]) * k.w[e] + k.b[e];
        activate(f, A.act);
    };
    float f[8];
    if (!c.mine) return;
#pragma unroll 1
    while (off + 8 <= t.lim) {
        const Chunk<DT> now = v;
        v = span_load<STREAM>(x, t, off + t.step);
        result(now, f);
        if (STREAM) stream_store_whole<DT>(y + off, f);
        else store_whole<DT>(y + off, f);
        off += t.step;
    }
    if (V == 1 && off < t.lim) { result(load_chunk<DT>(x + off, t.lim - off), f); store_chunk<DT>(y + off, t.lim - off, f); }
}
// The result: x once more, out of the caches where it fits.  2 x 262144 x 128 bf16 42 us = 6.4 TB/s read and written (memory); 8 x 4096 x 320 11.0 us, of it ~1.6 the join: latency.
// part: the sums' partial pairs, joined by every workgroup for itself (the first of a slab writes the statistics down), or null: the statistics are there already
// (Waves per SIMD asked for, here, in k_map_sums and in k_slab_forward: the compiler's own choice took a register or two more and lost one of six, 1024 x 512 x 320 178 -> 214 us.)
template <int V, bool DROP, bool STREAM> __global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(DT == PLENREG_F32 || DROP ? 5 : 6, 8))) void k_map_apply(NormArgs A, MapPlan P, const double2 *part) {
    extern __shared__ double2 lds[];
    const Column c = my_column(P, blockIdx.y);
    const Span t = my_span(A, P, c, P.apply_rows);
    Draw d = {};
    if (DROP) d = make_draw(A.rng, A.site, A.cut);
#pragma unroll 1
    for (int64_t n = blockIdx.z; n < A.N; n += gridDim.z) 
        span_apply<V, DROP, STREAM>(A, P, d, c, t, n, [&]() -> const double2 * {
            if (!part) return A.stats + n * A.G;
            const bool writes = A.stats && blockIdx.x == 0 && blockIdx.y == 0;
            __syncthreads();
            join_slab(A, P, part + n * A.G * P.splits * P.col_blocks, [&](int g) { return group_shift<DROP>(A, d, n, g); }, [&](int g, float shift, double sum, double squares) {
                lds[g] = finish_stats(A, A.count, (double)shift, sum, squares);
                if (writes) A.stats[n * A.G + g] = lds[g];
            });
            __syncthreads();
            return lds;
        });
}

// backward: s1, s2 += the sums of dz and dz xh of a span of slab n, per virtual channel; k: the thread's constants, left for the caller
template <int V, bool DROP> __device__ __forceinline__ void span_back_sums(const NormArgs &A, const MapPlan &P, const Draw &d, const Column &c, const Span &t, int64_t n, Constants<V> &k, double (&s1)[8],
                                                                           double (&s2)[8]) {
    const T *x = (const T *)A.x + n * A.x_stride + t.base, *dy = (const T *)A.dy + n * A.dy_stride + t.base;
    int off = t.off;
    Chunk<DT> v, g;
    if (t.lim >= 8) { v = span_load(x, t, off); g = span_load(dy, t, off); }
    load_constants<V>(A, P, A.stats + n * A.G, c.col, k);
    const auto add = [&](const Chunk<DT> &cx, const Chunk<DT> &cg, int valid) {
        const Mask<DROP ? V : 0> m(d, n * A.size + t.base + off);
        float xh[8], dv[8], dz[8];
        unpack(cx, m, xh);
        unpack(cg, dv);
        normalise<V>(k, xh);
        back_activation(A, x + off, n, 8 * c.col, valid, m, xh, dv, k.w, k.b, dz);
#pragma unroll
        for (int e = 0; e < 8; e++) { s1[e] += (double)dz[e]; s2[e] += (double)(dz[e] * xh[e]); }
    };
    if (!c.mine) return;
#pragma unroll 1
    while (off + 8 <= t.lim) {
        const Chunk<DT> now = v, gnow = g;
        v = span_load(x, t, off + t.step); g = span_load(dy, t, off + t.step);
        add(now, gnow, 8);
        off += t.step;
    }
    // (of the part's other elements dy is zero)
    if (V == 1 && off < t.lim) add(load_chunk<DT>(x + off, t.lim - off), load_chunk<DT>(dy + off, t.lim - off), t.lim - off);
}
// the workgroup's channel sums over its slabs, to[0 / 1][C] = sums of dz xh, dz, written with the last slab; between two slabs they are in running[0 / 1][C], in 64 bits: a workgroup of a tensor of
// 2^31 slabs walks over thousands of them.  (Each thread reads its own words there; with one slab to a workgroup there are none.)
__device__ __forceinline__ void channel_sums(const double (&s1)[8], const double (&s2)[8], const NormArgs &A, const MapPlan &P, const Column &c, double2 *lds, float *to, double *running, bool first_time,
                                             bool last_time) {
    const int NT = blockDim.x, lanes = 1 << P.chan_log, lane = threadIdx.x & (lanes - 1);
    __syncthreads();
    if (c.mine)
#pragma unroll
        for (int e = 0; e < 8; e++) lds[e * NT + c.r * P.bcol + c.col - c.first] = double2{s2[e], s1[e]};
    __syncthreads();
    const int from = P.q_log ? 0 : 8 * c.first, last = P.q_log || 8 * (c.first + P.bcol) > A.C ? A.C : 8 * (c.first + P.bcol);
#pragma unroll 1
    for (int c8 = from; c8 < last; c8 += NT >> P.chan_log) {
        const int ch = c8 + (threadIdx.x >> P.chan_log);
        double s = 0.0, q = 0.0;
        if (ch < last)
#pragma unroll 2
            for (int i = lane; i < P.R << P.q_log; i += lanes) {
                const int r = i >> P.q_log, vc = (i - (r << P.q_log)) * A.C + ch, col = (vc >> 3) - c.first;
                if (col < 0 || col >= P.bcol || col + c.first >= P.ncol) continue;
                const double2 v = lds[(vc & 7) * NT + r * P.bcol + col];
                s += v.x; q += v.y;
            }
        lanes_sum2(s, q, P.chan_log);
        if (ch < last && lane == 0) {
            if (!first_time) { s += running[ch]; q += running[A.C + ch]; }
            if (last_time) { to[ch] = (float)s; to[A.C + ch] = (float)q; }
            else { running[ch] = s; running[A.C + ch] = q; }
        }
    }
}
// Backward, first launch: 4 x 1089 x 195 f16 11.9 us, of it two joins in LDS; per workgroup the channel sums (params[workgroup][2][C]), per split their w-weighted group sums (part[n][g][split][column block] = sum w dz, sum w dz xh), in 64
// bits.
template <int V, bool DROP> __global__ __launch_bounds__(512) void k_map_back_sums(NormArgs A, MapPlan P, double2 *part, float *params, double *running) {
    extern __shared__ double2 lds[];
    const Column c = my_column(P, blockIdx.y);
    const Span t = my_span(A, P, c, P.rows_per);
    // (column blocks of one position each have channels of their own, of several positions they share them)
    const int64_t row = P.q_log ? (int64_t)blockIdx.z * gridDim.y + blockIdx.y : blockIdx.z;
    Draw d = {};
    if (DROP) d = make_draw(A.rng, A.site, A.cut);
#pragma unroll 1
    for (int64_t n = blockIdx.z; n < A.N; n += gridDim.z) {
        double s1[8] = {}, s2[8] = {};
        Constants<V> k;
        span_back_sums<V, DROP>(A, P, d, c, t, n, k, s1, s2);
        if (params) {
            const int64_t at = (row * gridDim.x + blockIdx.x) * 2 * A.C;
            channel_sums(s1, s2, A, P, c, lds, params + at, running + at, n == blockIdx.z, n + gridDim.z >= A.N);
        }
        if (c.mine)
#pragma unroll
            for (int e = 0; e < 8; e++) { s1[e] *= (double)k.w[e]; s2[e] *= (double)k.w[e]; }
        const int64_t parts = (int64_t)P.splits * P.col_blocks;
        double2 *out = part + n * A.G * parts + blockIdx.x * P.col_blocks + blockIdx.y;
        join_groups<V>(s1, s2, A, P, c, lds, Nothing(), [&](int g, float, double a, double b) { out[g * parts] = double2{a, b}; });
    }
}
// second launch: the first workgroups join the splits of each (n, g) into {mean of w dz, mean of w dz xh}, the others the parameter gradients
__global__ __launch_bounds__(1024) void k_map_back_join(NormArgs A, int splits, const double2 *part, const float *params, int param_rows, int join_blocks, double2 *means, void *dw, void *db) {
    __shared__ double lds[64 * 17];
    if ((int)blockIdx.x >= join_blocks) { param_columns(A, params, param_rows, blockIdx.x - join_blocks, dw, db, lds); return; }
    for (int64_t item = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 6); item < A.N * A.G; item += (int64_t)join_blocks * 16) {
        const double2 t = join_splits(part + item * splits, splits);
        if ((threadIdx.x & 63) == 0) means[item] = double2{t.x * A.inv_count, t.y * A.inv_count};
    }
}
// dx of a span of slab n; ready() -> per group {sum of w dz, sum of w dz xh}, which times `scale` are the means
template <int V, bool DROP, bool STREAM, class F>
__device__ __forceinline__ void span_back_apply(const NormArgs &A, const MapPlan &P, const Draw &d, const Column &c, const Span &t, int64_t n, double scale, F ready) {
    const T *x = (const T *)A.x + n * A.x_stride + t.base, *dy = (const T *)A.dy + n * A.dy_stride + t.base;
    T *dx = (T *)A.out + n * A.size + t.base;
    int off = t.off;
    Chunk<DT> v, g;
    if (t.lim >= 8) { v = span_load<STREAM>(x, t, off); g = span_load<STREAM>(dy, t, off); }
    Constants<V> k;
    load_constants<V>(A, P, A.stats + n * A.G, c.col, k);
    float m1[V == 2 ? 1 : 8], m2[V == 2 ? 1 : 8];
    {
        const double2 *means = ready();
        Channel ch(A, 8 * c.col);
#pragma unroll
        for (int e = 0; e < (V == 2 ? 1 : 8); e++) { const double2 m = means[ch.g]; m1[e] = (float)(m.x * scale); m2[e] = (float)(m.y * scale); ch.next(A); }
    }
    const auto result = [&](const Chunk<DT> &cx, const Chunk<DT> &cg, int valid, float (&dz)[8]) {
        const Mask<DROP ? V : 0> m(d, n * A.size + t.base + off);
        float xh[8], dv[8];
        unpack(cx, m, xh);
        unpack(cg, dv);
        normalise<V>(k, xh);
        back_activation(A, x + off, n, 8 * c.col, valid, m, xh, dv, k.w, k.b, dz);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int i = V == 2 ? 0 : e;
            dz[e] = m.keep(e, k.rstd[i] * (dz[e] * k.w[e] - m1[i] - xh[e] * m2[i]));
        }
    };
    float f[8];
    if (!c.mine) return;
#pragma unroll 1
    while (off + 8 <= t.lim) {
        const Chunk<DT> now = v, gnow = g;
        v = span_load<STREAM>(x, t, off + t.step); g = span_load<STREAM>(dy, t, off + t.step);
        result(now, gnow, 8, f);
        if (STREAM) stream_store_whole<DT>(dx + off, f);
        else store_whole<DT>(dx + off, f);
        off += t.step;
    }
    if (V == 1 && off < t.lim) {
        result(load_chunk<DT>(x + off, t.lim - off), load_chunk<DT>(dy + off, t.lim - off), t.lim - off, f);
        store_chunk<DT>(dx + off, t.lim - off, f);
    }
}
// The gradient of x; 4 x 1089 x 195 f16 8.5 us with the joins, both passes of 8 x 4096 x 320 bf16 53 us.
// part: the sums' partial pairs, joined by every workgroup for itself, or null: the means are there already.  The first P.param_z slices of the grid join the parameter gradients.
template <int V, bool DROP, bool STREAM>
__global__ __launch_bounds__(512) void k_map_back_apply(NormArgs A, MapPlan P, const double2 *part, const double2 *means, const float *params, int param_rows, void *dw, void *db) {
    extern __shared__ double2 lds[];
    if ((int)blockIdx.z < P.param_z) {
        const int block = ((int)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x;
        if (block * 16 < 2 * A.C) param_columns(A, params, param_rows, block, dw, db, (double *)lds);
        return;
    }
    const Column c = my_column(P, blockIdx.y);
    const Span t = my_span(A, P, c, P.apply_rows);
    Draw d = {};
    if (DROP) d = make_draw(A.rng, A.site, A.cut);
#pragma unroll 1
    for (int64_t n = blockIdx.z - P.param_z; n < A.N; n += gridDim.z - P.param_z)
        span_back_apply<V, DROP, STREAM>(A, P, d, c, t, n, part ? A.inv_count : 1.0, [&]() -> const double2 * {
            if (!part) return means + n * A.G;
            __syncthreads();
            join_slab(A, P, part + n * A.G * P.splits * P.col_blocks, Nothing(), [&](int g, float, double s1, double s2) { lds[g] = double2{s1, s2}; });
            __syncthreads();
            return lds;
        });
}

// ---- slabs that one workgroup goes over by itself: the same passes in one launch, the second reading out of the nearer caches.
//      256 x 512 x 320 bf16: forward 45 us, both passes 123 (split 44 and 167); 8 x 32 x 320 forward 7.0 (8.2).  `lds`: the join's space, then G pairs.
template <int V, bool DROP> __global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(DT == PLENREG_F32 ? 4 : 5, 8))) void k_slab_forward(NormArgs A, MapPlan P) {
    extern __shared__ double2 lds[];
    double2 *groups = lds + blockDim.x * (V == 2 ? 1 : 8);
    const Column c = my_column(P, 0);
    const Span t = my_span(A, P, c, P.rows);
    Draw d = {};
    if (DROP) { d = make_draw(A.rng, A.site, A.cut); write_used(A); }
#pragma unroll 1
    for (int64_t n = blockIdx.y; n < A.N; n += gridDim.y) {
        double s[8] = {}, q[8] = {};
        span_sums<V, DROP, DROP>(A, d, c, t, n, lds, s, q);
        join_groups<V>(s, q, A, P, c, lds, [&](int g) { return group_shift<DROP>(A, d, n, g); }, [&](int g, float shift, double sum, double squares) {
            groups[g] = finish_stats(A, A.count, (double)shift, sum, squares);
            if (A.stats) A.stats[n * A.G + g] = groups[g];
        });
        __syncthreads();
        span_apply<V, DROP, false>(A, P, d, c, t, n, [&] { return groups; });
    }
}
template <int V, bool DROP> __global__ __launch_bounds__(512) void k_slab_backward(NormArgs A, MapPlan P, float *params, double *running) {
    extern __shared__ double2 lds[];
    double2 *groups = lds + blockDim.x * 8;
    const Column c = my_column(P, 0);
    const Span t = my_span(A, P, c, P.rows);
    Draw d = {};
    if (DROP) d = make_draw(A.rng, A.site, A.cut);
#pragma unroll 1
    for (int64_t n = blockIdx.y; n < A.N; n += gridDim.y) {
        double s1[8] = {}, s2[8] = {};
        {
            Constants<V> k;
            span_back_sums<V, DROP>(A, P, d, c, t, n, k, s1, s2);
            const int64_t at = (int64_t)blockIdx.y * 2 * A.C;
            if (params) channel_sums(s1, s2, A, P, c, lds, params + at, running + at, n == blockIdx.y, n + gridDim.y >= A.N);
#pragma unroll
            for (int e = 0; e < 8; e++) { s1[e] *= (double)k.w[e]; s2[e] *= (double)k.w[e]; }
        }
        join_groups<V>(s1, s2, A, P, c, lds, Nothing(), [&](int g, float, double a, double b) { groups[g] = double2{a, b}; });
        __syncthreads();
        span_back_apply<V, DROP, false>(A, P, d, c, t, n, A.inv_count, [&] { return groups; });
    }
}

// ---- launches
template <int V, bool DROP, bool STREAM> void row_forward_v(const NormArgs &a, const RowLaunch &r, hipStream_t s) {
    if (r.K == 1) k_row_forward<V, 1, 256, DROP, STREAM><<<r.grid, 256, 0, s>>>(a, r.P);
    else if (r.K == 2) k_row_forward<V, 2, 256, DROP, STREAM><<<r.grid, 256, 0, s>>>(a, r.P);
    else k_row_forward<V, 4, 256, DROP, STREAM><<<r.grid, 256, 0, s>>>(a, r.P);
}
void row_forward(const NormArgs &a, const RowLaunch &r, hipStream_t s) {
    if (a.D % 8) a.cut ? row_forward_v<0, true, false>(a, r, s) : row_forward_v<0, false, false>(a, r, s);
    else if (r.stream) a.cut ? row_forward_v<1, true, true>(a, r, s) : row_forward_v<1, false, true>(a, r, s);
    else a.cut ? row_forward_v<1, true, false>(a, r, s) : row_forward_v<1, false, false>(a, r, s);
}
template <int V, bool DROP, bool STREAM> void row_backward_v(const NormArgs &a, const RowLaunch &r, float *part, hipStream_t s) {
    if (r.K == 1) k_row_backward<V, 1, 512, DROP, STREAM><<<r.grid, 512, 0, s>>>(a, r.P, part);
    else k_row_backward<V, 2, 512, DROP, STREAM><<<r.grid, 512, 0, s>>>(a, r.P, part);
}
void row_backward(const NormArgs &a, const RowLaunch &r, float *part, hipStream_t s) {
    if (a.D % 8) a.cut ? row_backward_v<0, true, false>(a, r, part, s) : row_backward_v<0, false, false>(a, r, part, s);
    else if (r.stream) a.cut ? row_backward_v<1, true, true>(a, r, part, s) : row_backward_v<1, false, true>(a, r, part, s);
    else a.cut ? row_backward_v<1, true, false>(a, r, part, s) : row_backward_v<1, false, false>(a, r, part, s);
}
unsigned column_blocks(const NormArgs &a) { return (unsigned)((2 * (int64_t)a.C + 15) / 16); }
template <int V, bool STREAM> void wide_forward_v(const NormArgs &a, const WideLaunch &m, hipStream_t s) {
    if (a.cut) k_wide_forward<V, true, STREAM><<<m.grid, WIDE_NT, 0, s>>>(a);
    else k_wide_forward<V, false, STREAM><<<m.grid, WIDE_NT, 0, s>>>(a);
}
void wide_forward(const NormArgs &a, const WideLaunch &m, hipStream_t s) {
    if (a.D % 8) wide_forward_v<0, false>(a, m, s);
    else m.stream ? wide_forward_v<1, true>(a, m, s) : wide_forward_v<1, false>(a, m, s);
}
template <int V, bool STREAM> void wide_backward_v(const NormArgs &a, const WideLaunch &m, float *part, hipStream_t s) {
    if (part) {
        if (a.cut) k_wide_params<V, true><<<m.params, 256, 0, s>>>(a, part);
        else k_wide_params<V, false><<<m.params, 256, 0, s>>>(a, part);
    }
    if (a.cut) k_wide_backward<V, true, STREAM><<<m.grid, WIDE_NT, 0, s>>>(a);
    else k_wide_backward<V, false, STREAM><<<m.grid, WIDE_NT, 0, s>>>(a);
}
void wide_backward(const NormArgs &a, const WideLaunch &m, float *part, hipStream_t s) {
    if (a.D % 8) wide_backward_v<0, false>(a, m, part, s);
    else m.stream ? wide_backward_v<1, true>(a, m, part, s) : wide_backward_v<1, false>(a, m, part, s);
}
void params(const NormArgs &a, const float *part, int rows, void *dw, void *db, hipStream_t s) { k_row_params<<<column_blocks(a), 1024, 0, s>>>(a, part, rows, dw, db); }

bool one_group(const NormArgs &a) { return a.C % 8 == 0 && a.D % 8 == 0; }
template <int V, bool DROP> void map_forward_v(const NormArgs &a, const MapLaunch &m, double2 *part, hipStream_t s) {
    const size_t lds = (size_t)m.NT * (V == 2 ? 16 : 128);
    if (m.slab) { k_slab_forward<V, DROP><<<m.sums, m.NT, lds + a.G * 16, s>>>(a, m.P); return; }
    if (V == 2 || DROP || m.lean) k_map_sums<V, DROP, true><<<m.sums, m.NT, lds, s>>>(a, m.P, part);
    else k_map_sums<V, DROP, V == 2 || DROP><<<m.sums, m.NT, lds, s>>>(a, m.P, part);
    if (!m.joins) k_map_stats<DROP><<<m.stat_blocks, 256, 0, s>>>(a, m.P.splits * m.P.col_blocks, part);
    const size_t stats = m.joins ? (size_t)a.G * 16 : 0;
    const double2 *join = m.joins ? part : nullptr;
    if (m.stream) k_map_apply<V, DROP, true><<<m.apply, m.NT, stats, s>>>(a, m.P, join);
    else k_map_apply<V, DROP, false><<<m.apply, m.NT, stats, s>>>(a, m.P, join);
}
void map_forward(const NormArgs &a, const MapLaunch &m, double2 *part, hipStream_t s) {
    if (one_group(a)) a.cut ? map_forward_v<2, true>(a, m, part, s) : map_forward_v<2, false>(a, m, part, s);
    else a.cut ? map_forward_v<1, true>(a, m, part, s) : map_forward_v<1, false>(a, m, part, s);
}
template <int V, bool DROP> void map_backward_v(const NormArgs &a, const MapLaunch &m, double2 *part, double2 *means, float *sums, double *running, void *dw, void *db, hipStream_t s) {
    if (m.slab) {
        k_slab_backward<V, DROP><<<m.sums, m.NT, (size_t)m.NT * 128 + a.G * 16, s>>>(a, m.P, sums, running);
        if (sums) params(a, sums, m.param_rows, dw, db, s);
        return;
    }
    k_map_back_sums<V, DROP><<<m.sums, m.NT, (size_t)m.NT * 128, s>>>(a, m.P, part, sums, running);
    MapPlan P = m.P;
    dim3 grid = m.apply;
    size_t lds = 0;
    if (m.joins) {
        if (sums) {
            P.param_z = (int)((column_blocks(a) + grid.x * grid.y - 1) / (grid.x * grid.y));
            grid.z += P.param_z;
            lds = (size_t)(m.NT / 16) * 17 * 8;
        }
        if (lds < (size_t)a.G * 16) lds = (size_t)a.G * 16;
    } else {
        const int64_t items = a.N * a.G;
        const int join = (int)(items < 16 * 4096 ? (items + 15) / 16 : 4096);
        k_map_back_join<<<join + (sums ? column_blocks(a) : 0), 1024, 0, s>>>(a, m.P.splits * m.P.col_blocks, part, sums, m.param_rows, join, means, dw, db);
    }
    const double2 *join = m.joins ? part : nullptr;
    if (m.stream) k_map_back_apply<V, DROP, true><<<grid, m.NT, lds, s>>>(a, P, join, means, sums, m.param_rows, dw, db);
    else k_map_back_apply<V, DROP, false><<<grid, m.NT, lds, s>>>(a, P, join, means, sums, m.param_rows, dw, db);
}
void map_backward(const NormArgs &a, const MapLaunch &m, double2 *part, double2 *means, float *sums, double *running, void *dw, void *db, hipStream_t s) {
    if (one_group(a)) a.cut ? map_backward_v<2, true>(a, m, part, means, sums, running, dw, db, s) : map_backward_v<2, false>(a, m, part, means, sums, running, dw, db, s);
    else a.cut ? map_backward_v<1, true>(a, m, part, means, sums, running, dw, db, s) : map_backward_v<1, false>(a, m, part, means, sums, running, dw, db, s);
}

}  // namespace

const NormEntry &REG_ENTRY() {
    static const NormEntry e = {row_forward, row_backward, wide_forward, wide_backward, map_forward, map_backward, params};
    return e;
}
