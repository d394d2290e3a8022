// The scan's forward pass, for whole regions and for single rows. Formulas and layout: statescan.h.
//
// Work per row, channel and state: one 2^x (8.3 clocks of a SIMD), two products and a sum over states (2.5 to 4 each), and a share of a
// matrix instruction; per row and channel some forty instructions more for softplus, gate and addresses. Measured: 193 495 rows of 256 float channels
// with 16 states 248 us (817 MB; memory alone would take 172), 33 282 rows of 1024 bfloat16 in three long regions 124 + 165 us. That is 720 clocks of a SIMD
// per row and wave, where the instructions alone come to some 430 at the rates above: a third of the waves' time is issue, a third waits for its
// turn to issue, a third for memory and LDS.
#include "statescan.h"

namespace dbk {

// n rows from `row` on, the states in registers. OUT: the rows of Y are written; otherwise only the states move on, and `steps` adds up d.
// kept: null, or the block of states in front of the first row's chunk of 8; those in front of the next ones are written behind it.
// What two rows need comes from memory while the two before them are worked on; their weights then lie in the wave's `lds`.
template <typename T, int LG, int NS, bool OUT>
__device__ __forceinline__ void scan_rows(const scan_shape& p, const scan_lane& l, unsigned lane, unsigned first, size_t row, unsigned n, const T* X, const T* dt, const T* gate,
                                          const typename acc_of<T>::type* B, const typename acc_of<T>::type* C, typename acc_of<T>::type skip,
                                          typename acc_of<T>::type bias, typename acc_of<T>::type (&h)[NS], const typename acc_of<T>::type (&k)[NS],
                                          T* Y, typename acc_of<T>::type* kept, typename acc_of<T>::type& steps, typename acc_of<T>::type* lds)
{
    typedef typename acc_of<T>::type A;
    constexpr int U = SCAN_AHEAD;
    typedef scan_weights<A, LG, NS, true, OUT> weights;
    if (!n) return;
    const unsigned at = opaque(l.ch * (unsigned)sizeof(T));
    T xn[U], dn[U], gn[U];
    weights w(p, lane, first, B + row * p.ldb, C + row * p.ldc, lds, 0u, false);
    const T *xp = X + row * p.ldx, *dp = dt + row * p.lddt, *gp = gate + row * p.ldg;
    T* yp = Y + row * p.ldy;
    auto fetch = [&](unsigned left) {            // (a row behind the last one: the last one again)
#pragma unroll
        for (int i = 0; i < U; ++i) {
            xn[i] = lane_load(xp, at);
            dn[i] = lane_load(dp, at);
            if (OUT && gate) gn[i] = lane_load(gp, at);
            const bool more = i + 1u < left;
            xp += more ? p.ldx : 0;
            dp += more ? p.lddt : 0;
            gp += more ? p.ldg : 0;
        }
        w.fetch(left);
    };
    fetch(n);
    for (unsigned t = 0; t < n; t += U) {
        A d[U], x[U];
        T g[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            A slope;
            x[i] = (A)xn[i];
            d[i] = step_of(p, (A)dn[i] + bias, slope);
            g[i] = gn[i];
        }
        w.put();
        if (t + U < n) fetch(n - t - U);
        if (OUT && kept && t && t % SCAN_CHUNK == 0) regs_to(p, l, h, kept + (size_t)(t / SCAN_CHUNK) * p.S * p.D);
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (t + i >= n) break;
            const A in = d[i] * x[i];
            A y[4] = {skip * x[i], A(0), A(0), A(0)};
            A bl[NS / 4];
            if constexpr (weights::MATRIX) w.b_of_lane(i, bl);
#pragma unroll
            for (int q = 0; q < NS; q += 4) {
                if constexpr (weights::MATRIX) {
                    A v[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[j] = exp2_fast(d[i] * k[q + j]) * h[q + j];
                    outer_add(v, bl[q / 4], in);
#pragma unroll
                    for (int j = 0; j < 4; ++j) h[q + j] = v[j];
                } else {
                    const quad<A> b = w.b(i, q);
#pragma unroll
                    for (int j = 0; j < 4; ++j) h[q + j] = fma_a(exp2_fast(d[i] * k[q + j]), h[q + j], in * b.v[j]);
                }
                if (OUT) {
                    const quad<A> c = w.c(i, q);
#pragma unroll
                    for (int j = 0; j < 4; ++j) y[j] = fma_a(c.v[j], h[q + j], y[j]);
                }
            }
            if (OUT) {
                A out = (y[0] + y[1]) + (y[2] + y[3]);
                if (gate) { const A gg = (A)g[i]; out *= gg * sigmoid_of(gg); }
                if (l.active) lane_store(yp, at, (T)out);
                yp += p.ldy;
            } else
                steps += d[i];
            __builtin_amdgcn_sched_barrier(0);   // (a row's work stays together: its operands would fill the registers with those of others)
        }
    }
}

// Four waves per SIMD, which float and bfloat16 rows with up to 16 states need no more than 89 of 128 registers for. More states, and doubles from 8 registers of states
// on, do not fit and spill: 2048 reads x 256 channels take 232 us with 16 float states, 556 with 32 and 3410 with 64, 2234 with 16 double ones.
// Blocks below nregion: a region, all of it or its first segment (the state behind which is carried to the second one); the
// others: what a segment makes of a zero state, where another one follows.
template <typename T, int LG, int NS>
__global__ __launch_bounds__(256, 4) void k_scan_fprop(scan_shape p, const uint32_t* __restrict__ regions, const uint32_t* __restrict__ marks,
                                                   const T* __restrict__ X, const T* __restrict__ dt,
                                                   const typename acc_of<T>::type* __restrict__ A_, const typename acc_of<T>::type* __restrict__ B,
                                                   const typename acc_of<T>::type* __restrict__ C, const typename acc_of<T>::type* __restrict__ skip,
                                                   const T* __restrict__ gate, const typename acc_of<T>::type* __restrict__ bias,
                                                   const typename acc_of<T>::type* __restrict__ state, T* __restrict__ Y,
                                                   typename acc_of<T>::type* __restrict__ last, typename acc_of<T>::type* __restrict__ keep,
                                                   typename acc_of<T>::type* __restrict__ local, typename acc_of<T>::type* __restrict__ sums,
                                                   typename acc_of<T>::type* __restrict__ carry)
{
    typedef typename acc_of<T>::type A;
    const unsigned tile = blockIdx.y * blockDim.y + uniform(threadIdx.y);
    if (tile >= p.tiles) return;
    __shared__ A lds_all[4][scan_weights<A, LG, NS, true, true>::SIZE];
    A* lds = lds_all[uniform(threadIdx.y)];
    const scan_lane l = lane_channel<LG>(p, tile, threadIdx.x);
    const unsigned first = first_group<LG>(p, tile);
    const size_t block = (size_t)p.S * p.D;
    const A sk = skip ? skip[l.ch] : A(0), bi = bias ? bias[l.ch] : A(0);
    A h[NS], a2[NS], steps = 0;
    if (blockIdx.x < p.nregion) {
        const unsigned r = blockIdx.x;
        const row_range g = region_rows(regions, r, p.N);
        const bool cut = marks && is_cut(p, g);
        regs_from(p, l, a2, A_, A(1.4426950408889634));
        regs_from(p, l, h, state ? state + (size_t)r * block : (const A*)nullptr, A(1));
        scan_rows<T, LG, NS, true>(p, l, threadIdx.x, first, g.start, cut ? p.seg : g.end - g.start, X, dt, gate, B, C, sk, bi, h, a2, Y,
                                         keep ? kept_at(p, keep, g.start, 0u) : (A*)nullptr, steps, lds);
        if (cut) regs_to(p, l, h, carry + (size_t)(g.start / p.seg + 1u) * block);
        else if (last) regs_to(p, l, h, last + (size_t)r * block);
        return;
    }
    unsigned r, k;
    row_range g;
    const unsigned slot = blockIdx.x - p.nregion;
    if (!cut_segment(p, regions, marks, slot, r, g, k) || g.start + (uint64_t)(k + 1u) * p.seg >= g.end) return;
    regs_from(p, l, a2, A_, A(1.4426950408889634));
    regs_from(p, l, h, (const A*)nullptr, A(1));
    scan_rows<T, LG, NS, false>(p, l, threadIdx.x, first, (size_t)g.start + (size_t)k * p.seg, p.seg, X, dt, gate, B, C, sk, bi, h, a2, Y, (A*)nullptr, steps, lds);
    regs_to(p, l, h, local + (size_t)slot * block);
    if (l.active) sums[(size_t)slot * p.D + l.ch] = steps;
}

// The state in front of every segment of a cut region from the one in front of the segment before: what that one makes of zeros, and
// its own carried state times exp(A * sum of its steps). A thread per state and channel.
template <typename A>
__global__ __launch_bounds__(256) void k_scan_carry(scan_shape p, const uint32_t* __restrict__ regions, const A* __restrict__ A_,
                                                    const A* __restrict__ local, const A* __restrict__ sums, A* __restrict__ carry)
{
    const row_range g = region_rows(regions, blockIdx.x, p.N);
    if (!is_cut(p, g)) return;
    const size_t block = (size_t)p.S * p.D, first = g.start / p.seg + 1u;
    const unsigned n = (g.end - g.start - 1u) / p.seg;             // segments behind the first; the state in front of the first of them is there
    for (size_t at = (size_t)blockIdx.y * 256u + threadIdx.x; at < block; at += (size_t)gridDim.y * 256u)
        carry_chain<A>(A_[at] * A(1.4426950408889634), carry[first * block + at], n - 1u, local + first * block + at, sums + first * p.D + at % p.D,
                       carry + (first + 1u) * block + at, block, p.D);
}

// The rows of every segment behind the first, from the state carried to it.
template <typename T, int LG, int NS>
__global__ __launch_bounds__(256, 4) void k_scan_fprop_cut(scan_shape p, const uint32_t* __restrict__ regions, const uint32_t* __restrict__ marks,
                                                       const T* __restrict__ X, const T* __restrict__ dt,
                                                       const typename acc_of<T>::type* __restrict__ A_, const typename acc_of<T>::type* __restrict__ B,
                                                       const typename acc_of<T>::type* __restrict__ C, const typename acc_of<T>::type* __restrict__ skip,
                                                       const T* __restrict__ gate, const typename acc_of<T>::type* __restrict__ bias, T* __restrict__ Y,
                                                       typename acc_of<T>::type* __restrict__ last, typename acc_of<T>::type* __restrict__ keep,
                                                       const typename acc_of<T>::type* __restrict__ carry)
{
    typedef typename acc_of<T>::type A;
    unsigned r, k;
    row_range g;
    if (!cut_segment(p, regions, marks, blockIdx.x, r, g, k)) return;
    const unsigned tile = blockIdx.y * blockDim.y + uniform(threadIdx.y);
    if (tile >= p.tiles) return;
    __shared__ A lds_all[4][scan_weights<A, LG, NS, true, true>::SIZE];
    A* lds = lds_all[uniform(threadIdx.y)];
    const scan_lane l = lane_channel<LG>(p, tile, threadIdx.x);
    const unsigned first = first_group<LG>(p, tile);
    const size_t block = (size_t)p.S * p.D;
    const A sk = skip ? skip[l.ch] : A(0), bi = bias ? bias[l.ch] : A(0);
    A h[NS], a2[NS], steps = 0, *kept = keep ? kept_at(p, keep, g.start, k * (p.seg / SCAN_CHUNK)) : (A*)nullptr;
    regs_from(p, l, a2, A_, A(1.4426950408889634));
    regs_from(p, l, h, carry + (size_t)blockIdx.x * block, A(1));
    if (kept) regs_to(p, l, h, kept);
    const unsigned row = g.start + k * p.seg;
    scan_rows<T, LG, NS, true>(p, l, threadIdx.x, first, row, min(p.seg, g.end - row), X, dt, gate, B, C, sk, bi, h, a2, Y, kept, steps, lds);
    if (last && g.end - row <= p.seg) regs_to(p, l, h, last + (size_t)r * block);
}

__global__ __launch_bounds__(256) void k_mark_cut(scan_shape p, const uint32_t* __restrict__ regions, uint32_t* __restrict__ marks)
{
    const unsigned r = blockIdx.x * 4u + (threadIdx.x >> 6);
    if (r >= p.nregion) return;
    const row_range g = region_rows(regions, r, p.N);
    if (is_cut(p, g)) mark_segments(marks, r, g, p.seg, threadIdx.x & 63u, 64u);
}
int mark_cut_regions(hipStream_t st, const scan_shape& p, const uint32_t* regions, uint32_t* marks)
{
    k_mark_cut<<<divup(p.nregion, 4), 256, 0, st>>>(p, regions, marks);
    return 0;
}

// One new row per sequence: four waves share a tile of 64 channels, a quarter of the states each.
template <typename T>
__global__ __launch_bounds__(256) void k_scan_step(scan_shape p, const T* __restrict__ X, const T* __restrict__ dt, const typename acc_of<T>::type* __restrict__ A_,
                                                   const typename acc_of<T>::type* __restrict__ B, const typename acc_of<T>::type* __restrict__ C,
                                                   const typename acc_of<T>::type* __restrict__ skip, const T* __restrict__ gate,
                                                   const typename acc_of<T>::type* __restrict__ bias, const typename acc_of<T>::type* state,
                                                   typename acc_of<T>::type* into, T* __restrict__ Y)
{
    typedef typename acc_of<T>::type A;
    __shared__ A sums[4][64];
    const unsigned lane = threadIdx.x & 63u, part = threadIdx.x >> 6, ch = blockIdx.y * 64u + lane;
    const size_t r = blockIdx.x;
    const bool active = ch < p.D;
    A y = 0, x = 0;
    if (active) {
        A slope;
        x = (A)X[r * p.ldx + ch];
        const A d = step_of(p, (A)dt[r * p.lddt + ch] + (bias ? bias[ch] : A(0)), slope), in = d * x;
        const unsigned group = ch / p.gs, per = (p.S + 3u) / 4u;
        const A *b = B + r * p.ldb + (size_t)group * p.S, *c = C + r * p.ldc + (size_t)group * p.S;
        const unsigned stop = min(p.S, (part + 1u) * per);
#pragma unroll 4
        for (unsigned s = part * per; s < stop; ++s) {
            const size_t at = (r * p.S + s) * p.D + ch;
            const A h = fma_a(exp2_fast(d * (A_[(size_t)s * p.D + ch] * A(1.4426950408889634))), state[at], in * b[s]);
            into[at] = h;
            y = fma_a(c[s], h, y);
        }
    }
    sums[part][lane] = y;
    __syncthreads();
    if (part || !active) return;
    y = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
    y = fma_a(skip ? skip[ch] : A(0), x, y);
    if (gate) { const A g = (A)gate[r * p.ldg + ch]; y *= g * sigmoid_of(g); }
    Y[r * p.ldy + ch] = (T)y;
}

namespace {

constexpr size_t SCAN_WAVES = 4096;              // waves that keep the vector units busy: four per SIMD (81 to 89 registers a lane, 16 float states, allow five)
constexpr size_t SCAN_LEAST = 32;                // rows of the shortest segment: its state's way through the carry costs as much as some ten rows

scan_plan plan_fprop(const dbk_statescan_args& a) { return plan_scan(a.N, a.D, a.G, SCAN_WAVES, 4, SCAN_LEAST); }

}  // namespace
}  // namespace dbk

using namespace dbk;

extern "C" {

int dbk_statescan_args_size(void) { return (int)sizeof(dbk_statescan_args); }

int dbk_statescan_workspace(const dbk_statescan_args* a, int backward, size_t* work_bytes)
{
    if (int rc = check_scan(a)) return rc;
    DBK_CHECK(work_bytes, "ValueError: null result");
    *work_bytes = 0;
    if (a->N && a->D && a->nregion) *work_bytes = backward ? bprop_work_bytes(*a) : segments_in(nullptr, *a, plan_fprop(*a)).bytes;
    clear_error();
    return 0;
}

int dbk_statescan(dbk_stream_t stream, const dbk_statescan_args* a, void* work, size_t work_bytes)
{
    if (int rc = check_scan(a)) return rc;
    DBK_CHECK(!a->nregion || a->regions, "ValueError: null regions");
    DBK_CHECK(!a->N || !a->D || a->Y, "ValueError: null matrix");
    DBK_CHECK(a->N <= 1 || a->ldy >= a->D, "ValueError: row strides must be at least the number of columns");
    DBK_CHECK(!a->keep || !a->state, "ValueError: states are kept for the backward pass of whole sequences, which starts from zeros: no initial state");
    if (!a->D || !a->nregion) { clear_error(); return 0; }
    const scan_plan p = plan_fprop(*a);
    const scan_segments g = segments_in(work, *a, p);
    DBK_CHECK(!g.bytes || (work && work_bytes >= g.bytes), "ValueError: the workspace has %zu bytes, %zu are needed", work_bytes, g.bytes);
    DBK_CHECK(grid_fits(a->nregion + p.slots, 256), "ValueError: map too large (%zu rows, %zu regions)", a->N, a->nregion);
    const scan_shape s = shape_of(*a, p);
    hipStream_t st = as_stream(stream);
    const unsigned waves = p.tpg < 4 ? (p.tpg ? p.tpg : 1u) : 4u;
    if (p.slots) mark_cut_regions(st, s, a->regions, g.marks);
    with_row_type(a->dtype, [&](auto t) {
        typedef decltype(t) T;
        typedef typename acc_of<T>::type A;
        with_lanes(p.lanes, [&](auto lanes) {
            with_states(a->S, [&](auto ns) {
                k_scan_fprop<T, lanes.value, ns.value><<<dim3((unsigned)a->nregion + p.slots, divup(p.tiles, waves)), dim3(64, waves), 0, st>>>(
                    s, a->regions, g.marks, (const T*)a->X, (const T*)a->dt, (const A*)a->A, (const A*)a->B, (const A*)a->C, (const A*)a->skip, (const T*)a->gate,
                    (const A*)a->dt_bias, (const A*)a->state, (T*)a->Y, (A*)a->last, (A*)a->keep, (A*)g.local, (A*)g.steps, (A*)g.carry);
                if (!p.slots) return;
                k_scan_carry<A><<<dim3((unsigned)a->nregion, carry_blocks(*a)), 256, 0, st>>>(s, a->regions, (const A*)a->A, (const A*)g.local, (const A*)g.steps,
                                                                                              (A*)g.carry);
                k_scan_fprop_cut<T, lanes.value, ns.value><<<dim3(p.slots, divup(p.tiles, waves)), dim3(64, waves), 0, st>>>(
                    s, a->regions, g.marks, (const T*)a->X, (const T*)a->dt, (const A*)a->A, (const A*)a->B, (const A*)a->C, (const A*)a->skip, (const T*)a->gate,
                    (const A*)a->dt_bias, (T*)a->Y, (A*)a->last, (A*)a->keep, (const A*)g.carry);
            });
        });
    });
    DBK_LAUNCH_OK();
}

int dbk_statescan_step(dbk_stream_t stream, const dbk_statescan_args* a)
{
    if (int rc = check_scan(a)) return rc;
    DBK_CHECK(!a->N || !a->D || (a->Y && a->state && a->last), "ValueError: null matrix or state");
    DBK_CHECK(a->N <= 1 || a->ldy >= a->D, "ValueError: row strides must be at least the number of columns");
    DBK_CHECK(grid_fits(a->N, 256), "ValueError: too many sequences (%zu)", a->N);
    if (!a->N || !a->D) { clear_error(); return 0; }
    const scan_shape s = shape_of(*a, plan_scan(0, a->D, a->G, 1, 2, 1));
    hipStream_t st = as_stream(stream);
    with_row_type(a->dtype, [&](auto t) {
        typedef decltype(t) T;
        typedef typename acc_of<T>::type A;
        k_scan_step<T><<<dim3((unsigned)a->N, divup(a->D, 64)), 256, 0, st>>>(s, (const T*)a->X, (const T*)a->dt, (const A*)a->A, (const A*)a->B, (const A*)a->C,
                                                                             (const A*)a->skip, (const T*)a->gate, (const A*)a->dt_bias, (const A*)a->state, (A*)a->last, (T*)a->Y);
    });
    DBK_LAUNCH_OK();
}

}  // extern "C"
