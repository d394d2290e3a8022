// Selective state space scan along the rows of every region of a map: S states per channel that decay and take in the rows,
//
//   d = softplus(dt + bias) (or dt),  h[t] = exp(d A) h[t-1] + d x B[t],  y = C[t] . h[t] + D x,  y *= g sigmoid(g)
//
// with A (S, channels) per channel, B and C per row and group of channels. Backward, with e = dy g sigmoid(g) and the gradient g[t] of h[t]
// running from the last row to the first:
//
//   g[t] = C e + a[t+1] g[t+1],  dx = d (B . g) + D e,  dd = x (B . g) + sum_s g a h[t-1] A,  dA = sum_t g a h[t-1] d,
//   dB = sum over the group's channels of g d x,  dC = the same of e h,  dD = sum_t e x,  ddt = dd sigmoid(dt + bias),  dbias = sum_t ddt
//
// A lane is a channel and a wave a tile of 64 channels, which walks down a region's rows with the states in registers; B and C, which the lanes of a
// group share, come through LDS. States are float32 (double for double rows).
#pragma once
#include <type_traits>
#include "rows_common.h"

namespace dbk {

constexpr unsigned SCAN_CHUNK = 8;               // rows between two kept states

struct scan_shape {
    unsigned N, D, S, G, gs, nregion;            // rows, channels, states, groups, channels per group, regions
    unsigned tpg, tiles, softplus;               // waves' tiles per group (64 lanes per group), or 0: several groups per wave; all tiles
    unsigned seg, cut;                           // rows per segment of a region that is cut; regions of more rows than `cut` are
    size_t ldx, lddt, ldb, ldc, ldg, ldy;
};

// The channel of a lane: LG = 64 lanes for the channels of one group (tpg tiles of 64), or LG lanes for each of 64 / LG groups.
struct scan_lane { unsigned group, ch; bool active; };
template <int LG> __device__ __forceinline__ scan_lane lane_channel(const scan_shape& p, unsigned tile, unsigned lane)
{
    scan_lane l;
    unsigned in;
    if (LG == 64) {
        l.group = tile / p.tpg;
        in = (tile - l.group * p.tpg) * 64u + lane;
        l.active = in < p.gs;
    } else {
        l.group = tile * (64u / LG) + lane / LG;
        in = lane % LG;
        l.active = l.group < p.G && in < p.gs;
        l.group = min(l.group, p.G - 1u);
    }
    l.ch = l.group * p.gs + min(in, p.gs - 1u);  // (a lane without a channel follows its group's last one and stores nothing)
    return l;
}

// A lane's element of a row: the row's address is the same in all lanes and stays in scalar registers, the lane's place is one 32-bit offset in
// bytes (D * 8 < 2^32). The compiler is told nothing about the offset (opaque): it would add it to every matrix' address beforehand, in two
// vector registers each, for as long as the kernel runs.
template <typename V> __device__ __forceinline__ V opaque(V v) { asm volatile("" : "+v"(v)); return v; }
template <typename T> __device__ __forceinline__ T lane_load(const T* row, unsigned bytes) { return *(const T*)((const char*)row + bytes); }
template <typename T> __device__ __forceinline__ void lane_store(T* row, unsigned bytes, T v) { *(T*)((char*)row + bytes) = v; }

__device__ __forceinline__ float fma_a(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ double fma_a(double a, double b, double c) { return fma(a, b, c); }

__device__ __forceinline__ float ldexp_a(float a, int e) { return ldexpf(a, e); }
__device__ __forceinline__ double ldexp_a(double a, int e) { return ldexp(a, e); }

template <typename A> __device__ __forceinline__ A step_of(const scan_shape& p, A raw, A& slope)
{
    if (p.softplus) return softplus_of(raw, slope);
    slope = A(1);
    return raw;
}

template <typename A> struct quad { A v[4]; } __attribute__((aligned(16)));

// v[j] += b_j x for four states j of every lane's channel x, where lane l of every four holds b_(l % 4) of its group: the 16 outer products of four by
// four that v_mfma_f32_4x4x1 forms, lanes being channels and registers states. One instruction beside the vector unit's work in
// place of four of it.
__device__ __forceinline__ void outer_add(float (&v)[4], float b, float x)
{
    typedef float f4 __attribute__((ext_vector_type(4)));
    const f4 s = __builtin_amdgcn_mfma_f32_4x4x1f32(b, x, (f4){v[0], v[1], v[2], v[3]}, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = s[j];
}

// The first of the groups that a wave's tile covers.
template <int LG> __device__ __forceinline__ unsigned first_group(const scan_shape& p, unsigned tile) { return LG == 64 ? tile / p.tpg : tile * (64u / LG); }

// Weights of two rows for a wave: fetched from memory into registers, a few per lane, put into LDS and read from there by the lanes of
// each group: [row][B, C][group of the wave][state]. They could come as scalar operands where a wave's
// channels are of one group, but a scalar load can not run far enough ahead of the rows: there are not the registers.
// From state S on, registers follow the last state that exists: the same decay, input and start. Where the states are summed (B and C both)
// they share its output, by halves: with n of them, 1/2, 1/4, ... 2^-n and 2^-n once more, which scale its C exactly. (With weights of zero in
// their place an infinite input would leave 0 * inf = NaN in them, and in every sum from then on.)
constexpr int SCAN_AHEAD = 2;
template <typename A, int LG, int NS, bool WITH_B, bool WITH_C> struct scan_weights {
    static constexpr bool MATRIX = WITH_B && sizeof(A) == 4;     // B for the matrix cores
    static constexpr bool SHARES = WITH_B && WITH_C;
    static constexpr int GW = 64 / LG, PART = GW * NS, ROW = PART * (WITH_B + WITH_C), SIZE = SCAN_AHEAD * ROW, PER = (SIZE + 63) / 64;
    const A *from[PER];
    size_t step[PER];
    bool here[PER];
    unsigned to[PER];
    int share[PER];                              // exponent of the share of C
    A next[PER];
    A *lds, *mine;
    unsigned lane;
    bool shared;                                 // some registers follow the last state
    // B and C at row `first_row` of the rows; back: from there towards the rows in front
    __device__ __forceinline__ scan_weights(const scan_shape& p, unsigned lane_, unsigned first, const A* B, const A* C, A* lds_, unsigned first_row, bool back)
        : lds(lds_), mine(lds_ + lane_ / LG * NS), lane(lane_ & 63u), shared(p.S < (unsigned)NS)
    {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const unsigned at = lane + 64u * i, in = at % ROW, g = in % PART / NS, s = in % NS;
            const bool c = WITH_C && in >= (WITH_B ? PART : 0);
            const size_t ld = c ? p.ldc : p.ldb;
            here[i] = at < SIZE && first + g < p.G;
            to[i] = MATRIX && !c ? at - s + s % 4u * (NS / 4) + s / 4u : at;
            from[i] = (c ? C : B) + (here[i] ? (first_row + at / ROW) * ld + (size_t)(first + g) * p.S + min(s, p.S - 1u) : 0);
            share[i] = c && s + 1u >= p.S ? -(int)min(s + 2u - p.S, (unsigned)NS - p.S) : 0;
            step[i] = back ? 0 - SCAN_AHEAD * ld : SCAN_AHEAD * ld;
        }
    }
    // the next SCAN_AHEAD rows, of which `left` exist
    __device__ __forceinline__ void fetch(unsigned left)
    {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            next[i] = here[i] && (lane + 64u * i) / ROW < left ? *from[i] : A(0);
            from[i] += step[i];
        }
    }
    __device__ __forceinline__ void put()
    {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (SHARES && shared) next[i] = ldexp_a(next[i], share[i]);
            if (SIZE % 64 == 0 || lane + 64u * i < SIZE) lds[to[i]] = next[i];
        }
        __builtin_amdgcn_wave_barrier();         // (one wave: LDS keeps its order)
    }
    __device__ __forceinline__ quad<A> b(int r, int q) const { return *(const quad<A>*)(mine + r * ROW + q); }
    // a lane's share of B where the matrix cores multiply it: state 4 q + lane % 4, one of its own four after another
    __device__ __forceinline__ void b_of_lane(int r, A (&v)[NS / 4]) const
    {
#pragma unroll
        for (int q = 0; q < NS / 4; ++q) v[q] = mine[r * ROW + (lane % 4u) * (NS / 4) + q];
    }
    __device__ __forceinline__ quad<A> c(int r, int q) const { return *(const quad<A>*)(mine + r * ROW + (WITH_B ? PART : 0) + q); }
};

// the states of a lane's channel between registers and (S, D) memory; null: zeros; behind the last one, that one again
template <typename A, int NS> __device__ __forceinline__ void regs_from(const scan_shape& p, const scan_lane& l, A (&h)[NS], const A* from, A scale)
{
    const unsigned at = opaque(l.ch * (unsigned)sizeof(A));
#pragma unroll
    for (int j = 0; j < NS; ++j) h[j] = from ? lane_load(from + (size_t)min((unsigned)j, p.S - 1u) * p.D, at) * scale : A(0);
}
template <typename A, int NS> __device__ __forceinline__ void regs_to(const scan_shape& p, const scan_lane& l, const A (&h)[NS], A* to)
{
    const unsigned at = opaque(l.ch * (unsigned)sizeof(A));
    if (!l.active) return;
#pragma unroll
    for (int j = 0; j < NS; ++j) if (j < (int)p.S) lane_store(to + (size_t)j * p.D, at, h[j]);
}

template <typename A> __device__ __forceinline__ A* kept_at(const scan_shape& p, A* keep, unsigned start, unsigned chunk)
{
    return keep + ((size_t)start / SCAN_CHUNK + chunk) * p.S * p.D;
}

constexpr unsigned SCAN_STATES = 64;             // the most states per channel

// Lanes per group and tiles of channels; rows per segment, rows from which on a region is cut, and segment slots (0: none can be).
struct scan_plan { int lanes; unsigned tpg, tiles, seg, cut, slots; };

// A region is one wave's work, until it is so long that the others wait for it: then it is cut into segments. The segments' states are first
// found from zeros (a second pass over the rows, with three more launches), carried over from segment to segment, and the rows
// then written with the right states in front. The segment is an even share of all rows for `waves` waves, and a region is cut
// from `shares` of them on, but never one of up to 128 rows: 17 sequences of up to 77 double rows took 435 us both ways cut into segments of 32, 299 whole.
// (One line for all types: a wave walks 77 rows of five double states in some 100 us, of floats in a fraction of that; the four launches take 20.)
inline scan_plan plan_scan(size_t N, size_t D, size_t G, size_t waves, size_t shares, size_t least)
{
    scan_plan p;
    const size_t gs = D / G;
    p.lanes = gs <= 16 ? 16 : gs <= 32 ? 32 : 64;
    p.tpg = p.lanes == 64 ? divup(gs, 64) : 0u;
    p.tiles = p.lanes == 64 ? (unsigned)(G * p.tpg) : divup(G, 64 / p.lanes);
    const size_t share = (N * p.tiles / waves + SCAN_CHUNK - 1) / SCAN_CHUNK * SCAN_CHUNK;
    const size_t seg = share > least ? share : least, most = size_t(1) << 28;
    p.seg = (unsigned)(seg < most ? seg : most);
    p.cut = (unsigned)(p.seg * shares > 128 ? p.seg * shares : 128);
    p.slots = N > p.cut ? (unsigned)segment_slots(N, p.seg) : 0u;
    return p;
}

inline scan_shape shape_of(const dbk_statescan_args& a, const scan_plan& p)
{
    scan_shape s;
    s.N = (unsigned)a.N; s.D = (unsigned)a.D; s.S = (unsigned)a.S; s.G = (unsigned)a.G; s.gs = (unsigned)(a.D / a.G); s.nregion = (unsigned)a.nregion;
    s.tpg = p.tpg; s.tiles = p.tiles; s.seg = p.seg; s.cut = p.cut; s.softplus = a.softplus != 0;
    s.ldx = a.ldx; s.lddt = a.lddt; s.ldb = a.ldb; s.ldc = a.ldc; s.ldg = a.ldgate; s.ldy = a.ldy;
    return s;
}

template <typename F> void with_lanes(int lanes, F f)
{
    if (lanes == 16) f(std::integral_constant<int, 16>());
    else if (lanes == 32) f(std::integral_constant<int, 32>());
    else f(std::integral_constant<int, 64>());
}

// Registers for the states.
template <typename F> void with_states(size_t S, F f)
{
    if (S <= 4) f(std::integral_constant<int, 4>());
    else if (S <= 8) f(std::integral_constant<int, 8>());
    else if (S <= 16) f(std::integral_constant<int, 16>());
    else if (S <= 32) f(std::integral_constant<int, 32>());
    else f(std::integral_constant<int, 64>());
}

inline int check_scan(const dbk_statescan_args* a)
{
    DBK_CHECK(a, "ValueError: null argument block");
    DBK_ROW_DTYPE_OK(a->dtype);
    DBK_CHECK(a->S >= 1 && a->S <= SCAN_STATES, "NotImplementedError: 1 to %u states per channel, got %zu", SCAN_STATES, a->S);
    DBK_CHECK(a->G >= 1 && a->D % a->G == 0, "ValueError: the number of channels must be divisible by the number of groups");
    DBK_CHECK(a->N < (size_t(1) << 32) - 64 && a->D < (size_t(1) << 21) && a->nregion < (size_t(1) << 31), "ValueError: map too large (%zu rows, %zu channels, %zu regions)",
              a->N, a->D, a->nregion);
    DBK_CHECK(!a->D || a->A, "ValueError: null weights");
    DBK_CHECK(!a->N || !a->D || (a->X && a->dt && a->B && a->C), "ValueError: null matrix");
    DBK_CHECK(a->N <= 1 || (a->ldx >= a->D && a->lddt >= a->D && a->ldb >= a->G * a->S && a->ldc >= a->G * a->S && (!a->gate || a->ldgate >= a->D)),
              "ValueError: row strides must be at least the number of columns");
    DBK_CHECK(plan_scan(0, a->D, a->G, 1, 2, 1).tiles <= 65535u, "ValueError: too many groups (%zu of %zu channels)", a->G, a->G ? a->D / a->G : 0);
    return 0;
}

// The segments of a call's long regions, in its workspace: marks (one per slot), what the segments leave from zeros, the sums of
// their steps, and the states in front of them.
struct scan_segments { uint32_t* marks; void *local, *steps, *carry; size_t bytes; };
inline scan_segments segments_in(void* work, const dbk_statescan_args& a, const scan_plan& p)
{
    scan_segments s;
    const size_t e = acc_size(a.dtype), states = (p.slots * a.S * a.D * e + 15) / 16 * 16;
    size_t at = ((size_t)p.slots * 4 + 15) / 16 * 16;
    s.marks = (uint32_t*)work;
    s.local = (char*)work + at;
    s.carry = (char*)work + (at += states);
    s.steps = (char*)work + (at += states);
    s.bytes = at + (p.slots * a.D * e + 15) / 16 * 16;
    if (!p.slots) { s.marks = nullptr; s.bytes = 0; }
    return s;
}

__device__ __forceinline__ bool is_cut(const scan_shape& p, row_range g) { return g.end - g.start > p.cut; }
__device__ __forceinline__ bool cut_segment(const scan_shape& p, const uint32_t* regions, const uint32_t* marks, unsigned slot, unsigned& r, row_range& g, unsigned& k)
{
    return slot_segment(regions, p.nregion, p.N, marks, slot, p.seg, r, g, k) && is_cut(p, g);
}
size_t bprop_work_bytes(const dbk_statescan_args& a);            // statescan_bprop.hip
// One state's way through n segments: s = local + exp2(a2 * sum) s after each, written to out; the three pointers start at the first and move
// on by `step` (sums by `sum_step`). U segments' values are on their way while U others are worked on.
// The factor comes in two halves: it may overflow or underflow where the product, which rows would form step by step, does not. A half is kept to what
// a normal number holds, so that nothing times the most growth is nothing, and an infinite state times the most decay still infinite. That changes growth
// by more than 2^254 (float), which overflows from any normal number, and decay by more than 2^252, which leaves less than 2^-124 of any.
template <typename A> __device__ __forceinline__ A half_power(A x)
{
    constexpr A up = sizeof(A) == 8 ? A(1023) : A(127), down = A(1) - up;
    return exp2_fast(x > up ? up : x < down ? down : x);        // (a NaN stays)
}
template <typename A> __device__ __forceinline__ void carry_chain(A a2, A s, unsigned n, const A* local, const A* sums, A* out, size_t step, size_t sum_step)
{
    constexpr unsigned U = 8;
    A add[U], sum[U];
    auto fetch = [&](unsigned left) {
#pragma unroll
        for (unsigned i = 0; i < U; ++i) {
            add[i] = *local;
            sum[i] = *sums;
            local += i + 1u < left ? step : 0;
            sums += i + 1u < left ? sum_step : 0;
        }
    };
    if (!n) return;
    fetch(n);
    for (unsigned k = 0; k < n; k += U) {
        A av[U], sv[U];
#pragma unroll
        for (unsigned i = 0; i < U; ++i) { av[i] = add[i]; sv[i] = half_power(A(0.5) * a2 * sum[i]); }
        if (k + U < n) fetch(n - k - U);
#pragma unroll
        for (unsigned i = 0; i < U; ++i) {
            if (k + i >= n) break;
            s = fma_a(sv[i], sv[i] * s, av[i]);
            *out = s;
            out += step;
        }
    }
}
// workgroups per region for the carries: few regions share the chip, many take little of it each
inline unsigned carry_blocks(const dbk_statescan_args& a)
{
    const size_t need = (a.S * a.D + 255) / 256, room = 2048 / a.nregion + 1;
    return (unsigned)(need < room ? need : room);
}

// marks the segments behind the first of every region that is cut: a wave per region
int mark_cut_regions(hipStream_t st, const scan_shape& p, const uint32_t* regions, uint32_t* marks);

}  // namespace dbk
