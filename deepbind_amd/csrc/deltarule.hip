// The gated delta rule's forward pass, for whole regions and for single rows. Formulas and layout: deltarule.h.
#include "deltarule.h"

namespace dbk {

__global__ __launch_bounds__(256) void k_delta_mark(delta_shape p, const uint32_t* __restrict__ regions, uint32_t* __restrict__ marks, uint32_t* __restrict__ cuts, uint32_t* __restrict__ odd)
{
    // a wave per region
    const unsigned r = blockIdx.x * 4u + (threadIdx.x >> 6);
    if (r >= p.nregion) return;
    const row_range g = region_rows(regions, r, p.N);
    mark_segments(marks, r, g, DELTA_BLOCK, threadIdx.x & 63u, 64u);
    if (p.L) mark_segments(cuts, r, g, p.L, threadIdx.x & 63u, 64u);
    for (unsigned h = threadIdx.x & 63u; h < p.H; h += 64u) odd[(size_t)r * p.H + h] = 0u;
    if (blockIdx.x == 0u && threadIdx.x == 0u) odd[(size_t)p.nregion * p.H] = 0u;
}

// A chunk's matrices. A wave takes a block of a head, four chunks: the products of its keys and queries on the matrix cores, then a lane per chunk and column for the
// decays between rows and the triangle's inverse, column by column by substitution (powers of the triangle, which the matrix cores
// could multiply instead, grow far beyond the inverse where keys come again, and lose it). A wave waits for memory most of its time, first for its block, then for its
// rows: what it needs is asked for at once, and keys' products and queries' use its share of LDS in turn. Five waves run per SIMD with keys of up to 32 columns (bfloat16: 64), three with 64 floats
// or 128 bfloat16 values, two with 128 floats: as many as their registers allow. 191 284 rows in 2048 regions, 4 heads of
// 64 floats: 108 us for 460 MB (keys and queries in, matrices out; 90 at a copy's rate); 48 532 rows of 24 heads of 16, where four waves share a row's line: 84 us for 306 MB
// forward and 390 backward (106 with a square for each triangle).
template <typename T, int KT>
__global__ __launch_bounds__(256, (sizeof(T) < 8 && sizeof(T) * KT <= 8 ? 5 : 1)) void k_delta_prepare(delta_shape p, const uint32_t* __restrict__ regions, const uint32_t* __restrict__ marks, const T* __restrict__ Q,
                                                       const T* __restrict__ K, const typename acc_of<T>::type* __restrict__ beta,
                                                       const typename acc_of<T>::type* __restrict__ decay, delta_chunk<typename acc_of<T>::type>* __restrict__ chunks,
                                                       delta_pairs<typename acc_of<T>::type>* __restrict__ pairs, uint32_t* __restrict__ odd)
{
    typedef typename acc_of<T>::type A;
    typedef typename mm16<A>::vec vec;
    __shared__ __align__(16) A lds_all[4][4][16][20];
    __shared__ double a_all[4][64];
    __shared__ A b_all[4][64];
    const unsigned wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63u, g = lane >> 4, c = lane & 15u;
    A (*lds)[16][20] = lds_all[wave];
    A* b = b_all[wave];
    double* a = a_all[wave];
    delta_block bl;
    if (!find_block(p, regions, marks, blockIdx.x, bl)) return;
    const unsigned head = min(blockIdx.y * 4u + wave, p.H - 1u), group = head / (p.H / p.G);      // (a wave too many does the last head again)
    const unsigned nchunk = (bl.rows + 15u) / 16u;
    // two chunks' tiles are on their way at a time, in turn
    delta_tiles<T, KT> k[2], q[2];
    auto fetch = [&](unsigned i, int to) {
        const size_t row = bl.at + 16u * i;
        const unsigned rows = bl.rows - 16u * i;
        k[to].fetch(K + row * p.ldk + (size_t)group * p.K, p.ldk, rows, p.K, g, c);
        q[to].fetch(Q + row * p.ldq + (size_t)group * p.K, p.ldq, rows, p.K, g, c);
    };
    fetch(0u, 0);
    raw_one<A> rate, step;
    {
        const size_t row = bl.at + min(lane, bl.rows - 1u);
        step.load(beta + row * p.ldb + head);
        rate.load(decay ? decay + row * p.ldg + head : beta + row * p.ldb + head);
    }
    vec ms[DELTA_CHUNKS], ss[DELTA_CHUNKS];
#pragma unroll
    for (int i = 0; i < (int)DELTA_CHUNKS; ++i) {
        ms[i] = ss[i] = zero16<A>();
        if (i >= (int)nchunk) continue;
        if (i + 1 < (int)nchunk) fetch(i + 1u, (i + 1) & 1);
        const unsigned rows = bl.rows - 16u * i;
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            const vec kt = k[i & 1].get(t, rows, p.K, g, c), qt = q[i & 1].get(t, rows, p.K, g, c);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                ms[i] = mm16<A>::mac(kt[r], kt[r], ms[i]);
                ss[i] = mm16<A>::mac(qt[r], kt[r], ss[i]);
            }
        }
    }
    auto sync = []() { team_sync<1>(); };        // (a wave's LDS is its own)
    auto put = [&](const vec (&x)[DELTA_CHUNKS]) {
#pragma unroll
        for (int i = 0; i < (int)DELTA_CHUNKS; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) lds[i][mm16<A>::row(g, r)][c] = x[i][r];
        sync();
    };
    // two triangles of every chunk through LDS to memory, as a square of 16 x 16 values, consecutive lanes to consecutive places: what is below lies at [c][row], what is
    // above at [row][c]
    auto number = [&](unsigned i) { return chunk_number(p, bl.r, bl.g.start, bl.k * DELTA_CHUNKS + i, head); };
    auto store = [&](auto matrix, const A (&below)[16], const A (&above)[16]) {
        sync();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (i >= (int)c) lds[g][c][i] = below[i];
            if (i > (int)c) lds[g][i][c] = above[i];
        }
        sync();
        for (unsigned i = 0; i < nchunk; ++i) {
            row_vec<A, 4> v;
#pragma unroll
            for (int j = 0; j < 4; ++j) v.v[j] = lds[i][lane >> 2][4u * (lane & 3u) + j];
            v.store(matrix(number(i)) + 4u * lane, 4u);
        }
        sync();
    };
    put(ms);
    a[lane] = decay && lane < bl.rows ? exp((double)rate.get(true)) : 1.0;
    b[lane] = step.get(lane < bl.rows);
    sync();
    // lane (g, c): column c of chunk g
    A D[16], n[16], finite = A(0), size = A(0);
    {
        // (in double precision: a state that decays by a thousandth a row remembers a thousand of them, and would their factors' roundings)
        double product = 0.0, first = 1.0;
        A mine = A(1);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const double ai = a[16u * g + i];
            product = i == (int)c ? 1.0 : product * ai;          // (zero above the diagonal: nothing there yet)
            D[i] = i >= (int)c ? (A)product : A(0);
            first *= ai;
            mine = i == (int)c ? (A)first : mine;
            n[i] = i > (int)c ? D[i] * lds[g][i][c] : A(0);
            size = fmax(size, D[i]);
        }
        size = fmax(size, mine);
        // (a key's product with itself is finite where it is, and then those with all others are)
        finite = fma((A)a[16u * g + c], A(0), fma(b[16u * g + c], A(0), lds[g][c][c] * A(0)));
        // a row lengthens what lies along its key by the factor |1 - b k.k|, which lies within rounding's reach of one where keys of length one are learnt by b = 2
        const A turned = b[16u * g + c] * lds[g][c][c];
        if (__any(a[lane] > 1.0 || turned > A(2.05) || turned < A(-0.05)) && lane == 0u) atomicOr(odd + (size_t)bl.r * p.H + head, DELTA_GROWS);
        if (__any(a[lane] > 1.0)) {              // (does a product that is almost nothing grow again)
            product = 0.0;
            first = 1.0;
#pragma unroll 1
            for (unsigned i = 0; i < 16u; ++i) {
                const double ai = a[16u * g + i];
                if (ai > 1.0 && ((product > 0.0 && product < delta_range<A>::least) || (first > 0.0 && first < delta_range<A>::least))) size = A(INFINITY);
                product = i == c ? 1.0 : product * ai;
                first *= ai;
            }
        }
        if (g < nchunk) {
            delta_chunk<A>& to = chunks[number(g)];
            to.first[c] = mine;
            to.last[c] = D[15];
            to.b[c] = b[16u * g + c];
        }
    }
    if (pairs) store([&](size_t i) { return pairs[i].ND; }, n, D);
    sync();
#pragma unroll
    for (int i = 0; i < 16; ++i) lds[g][i][c] = n[i];
    sync();
    A x[16];
    // A column of the inverse is zero above its own row, and takes nothing from columns before it: where a value in them is not finite (zero times it would be a NaN, and
    // send one back to rows behind a bad key or decay, whose own gradients do not know of it) their places are left out one by one.
    auto substitute = [&](auto careful) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            A s[4] = {A(0), A(0), A(0), A(0)};
#pragma unroll
            for (int m = 0; m < i; ++m) s[m & 3] = careful.value && m < (int)c ? s[m & 3] : fma(lds[g][i][m], x[m], s[m & 3]);
            x[i] = i <= (int)c ? (i == (int)c ? A(1) : A(0)) : -b[16u * g + i] * ((s[0] + s[1]) + (s[2] + s[3]));
        }
    };
    substitute(std::false_type());
    A stray = A(0);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        stray = fma(x[i], A(0), stray);
        size = fmax(size, fabs(x[i]));
    }
    if (__any(stray != A(0))) substitute(std::true_type());
    const uint64_t beyond = __ballot(size > A(delta_range<A>::most)), bad = __ballot(finite != A(0));
    // (rarely any; the order in which marks are added does not matter)
    if (c == 0u && (beyond >> 16u * g & 0xffffu) && !(bad >> 16u * g & 0xffffu)) {
        atomicOr(odd + (size_t)bl.r * p.H + head, DELTA_ODD);
        odd[(size_t)p.nregion * p.H] = 1u;
    }
    sync();
    put(ss);
    A s[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = i >= (int)c ? D[i] * lds[g][i][c] : A(0);
    store([&](size_t i) { return chunks[i].TP; }, s, x);
}

// Walks a wave's 16 columns of a head's state down `rows` rows from `row` on, of region r, which starts at `first`.
// Keys, queries, matrices and values of a chunk come while the one before it is worked on. OUT: rows of O are written; otherwise only the state moves on. V null:
// without values, for what becomes of the state alone, whose columns are kept near one where they may grow (leveled; exponents in e). Bound by issue and by one chunk's chain, which waves of
// other heads and regions fill: 191 284 rows, 4 heads of 64 x 64 floats 293 us (850 MB at 2.9 TB/s, 23 GFLOP: matrix units busy for 51 % of the time, vector instructions 31 %); 41 816 bfloat16
// rows, 8 heads of 128 x 128 in 32 segments 249 us (28 % and 57 %, most of which takes the states apart into pieces). Four waves on the same head's keys share what is fetched: alone,
// each would read all of it.
template <typename T, int KT, int TEAM, bool OUT>
__device__ __forceinline__ void delta_walk(const delta_shape& p, const delta_lane<typename acc_of<T>::type, TEAM>& l, typename delta_ops<T, KT>::rows* lds, const T* Q, const T* K,
                                           const T* V, const delta_chunk<typename acc_of<T>::type>* chunks, typename acc_of<T>::type scale, unsigned r, unsigned first, size_t row, unsigned rows,
                                           typename mm16<typename acc_of<T>::type>::vec (&S)[KT], T* O, typename acc_of<T>::type* keep, size_t kept, bool leveled, int& e)
{
    typedef typename acc_of<T>::type A;
    typedef typename mm16<A>::vec vec;
    if (!rows) return;
    const T *q = Q + row * p.ldq + (size_t)l.group * p.K, *k = K + row * p.ldk + (size_t)l.group * p.K, *v = V + row * p.ldv + l.v;
    T* o = O + row * p.ldo + l.v + l.c;
    delta_feed<T, KT, TEAM, OUT> feed;
    const delta_chunk<A>* at = chunks + chunk_number(p, r, first, (unsigned)(row - first) / DELTA_CHUNK, l.head);
    auto fetch = [&](unsigned t) {
        feed.fetch(p, q + t * p.ldq, k + t * p.ldk, *at, l.thread, rows - t);
        at = t ? at + 1 : chunks + chunk_number(p, r, first, (unsigned)(row - first) / DELTA_CHUNK + 1u, l.head);
    };
    delta_values<T> values;
    fetch(0u);
    if (V) values.fetch(l, v, p.ldv, rows);
    feed.clear(lds[0].c, l.thread);
    feed.clear(lds[1].c, l.thread);
    feed.put(p, lds[0], l.thread);
    if (rows > DELTA_CHUNK) fetch(DELTA_CHUNK);
    team_sync<TEAM>();
    for (unsigned t = 0; t < rows; t += DELTA_CHUNK) {
        const unsigned n = min(rows - t, DELTA_CHUNK);
        const typename delta_ops<T, KT>::rows& here = lds[t / DELTA_CHUNK & 1u];
        vec x = V ? values.get(l) : zero16<A>();
        if (t + DELTA_CHUNK < rows) {
            feed.put(p, lds[~(t / DELTA_CHUNK) & 1u], l.thread);
            if (V) values.fetch(l, v + (t + DELTA_CHUNK) * p.ldv, p.ldv, rows - t - DELTA_CHUNK);
        }
        if (t + 2u * DELTA_CHUNK < rows) fetch(t + 2u * DELTA_CHUNK);
        if (l.nv) {
            if constexpr (!OUT)
                if (leveled) level<A, KT>(S, e);
            if (keep && (t || row != first) && t % DELTA_BLOCK == 0) store_state<A, KT>(S, keep + (kept + t / DELTA_BLOCK) * ((size_t)p.K * p.H * p.V), p, l);
            vec w = zero16<A>(), z = zero16<A>();
            delta_ops<T, KT>::template find<OUT>(here.k, here.q, S, w, z, l.g, l.c);
            const vec decayed = by_row(here.c.first, l.g), b = by_row(here.c.b, l.g);
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = l.row(r) < n ? b[r] * (x[r] - decayed[r] * w[r]) : A(0);
            const vec u = triangle<A, true>(matrix_by_rows(here.c.T, l.g, l.c), x, zero16<A>(), l.g);
            const vec sent = by_row(here.c.last, l.g) * u;
            const A through = here.c.first[15];
#pragma unroll
            for (int i = 0; i < KT; ++i) S[i] *= through;
            delta_ops<T, KT>::add(S, here.k, sent, l.g, l.c);
            if (OUT) {
                const vec y = triangle<A, true>(matrix_by_rows(here.c.P, l.g, l.c), u, decayed * z, l.g);
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (l.row(r) < n && l.c < l.nv) o[(size_t)(t + l.row(r)) * p.ldo] = (T)(scale * y[r]);
            }
        }
        team_sync<TEAM>();
    }
}

// A region of a marked head, row by row: 4096 rows of 16 heads of 64 x 64 floats 5.8 ms (by chunks 0.25), and 33 backward (0.33), as nothing is overlapped here.
template <typename T, int KT, int TEAM>
__device__ __forceinline__ void delta_walk_rows(const delta_shape& p, const delta_lane<typename acc_of<T>::type, TEAM>& l, const T* Q, const T* K, const T* V, const typename acc_of<T>::type* beta,
                                                const typename acc_of<T>::type* decay, typename acc_of<T>::type scale, row_range g, typename mm16<typename acc_of<T>::type>::vec (&S)[KT], T* O,
                                                typename acc_of<T>::type* keep)
{
    typedef typename acc_of<T>::type A;
    const bool here = l.c < l.nv;
#pragma unroll 1
    for (size_t row = g.start; row < g.end; ++row) {
        const unsigned at = (unsigned)row - g.start;
        if (keep && at && at % DELTA_BLOCK == 0) store_state<A, KT>(S, keep + kept_number(g, at / DELTA_BLOCK) * ((size_t)p.K * p.H * p.V), p, l);
        typename mm16<A>::vec x[KT];
        const A a = row_factor(p, decay, row, l.head);
        row_tiles<A, KT>(x, K + row * p.ldk + (size_t)l.group * p.K, p.K, l.g);
#pragma unroll
        for (int t = 0; t < KT; ++t) S[t] *= a;
        const A u = beta[row * p.ldb + l.head] * ((here ? (A)V[row * p.ldv + l.v + l.c] : A(0)) - found<A, KT>(x, S));
#pragma unroll
        for (int t = 0; t < KT; ++t) S[t] += x[t] * u;
        row_tiles<A, KT>(x, Q + row * p.ldq + (size_t)l.group * p.K, p.K, l.g);
        const A o = scale * found<A, KT>(x, S);
        if (here && l.g == 0u) O[row * p.ldo + l.v + l.c] = (T)o;
    }
}

// Workgroups below nregion: a region, or the first segment of a cut one; the others: the segment of their slot, from the state carried there. Of a marked head the first
// does the whole region (a kernel of their own for marked heads, behind this one, is a launch more: 30 us for 27 on a region of 63 rows).
template <typename T, int KT, int TEAM>
__global__ __launch_bounds__(256, (delta_waves<typename acc_of<T>::type, KT, TEAM>())) void k_delta_fprop(delta_shape p, const uint32_t* __restrict__ regions, const uint32_t* __restrict__ cuts,
                                                     const uint32_t* __restrict__ odd, const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V,
                                                     const typename acc_of<T>::type* __restrict__ beta, const typename acc_of<T>::type* __restrict__ decay,
                                                     const delta_chunk<typename acc_of<T>::type>* __restrict__ chunks, typename acc_of<T>::type scale,
                                                     const typename acc_of<T>::type* __restrict__ state, const typename acc_of<T>::type* __restrict__ carry, T* __restrict__ O,
                                                     typename acc_of<T>::type* __restrict__ last, typename acc_of<T>::type* __restrict__ keep)
{
    typedef typename acc_of<T>::type A;
    typedef typename mm16<A>::vec vec;
    __shared__ typename delta_ops<T, KT>::rows lds[4 / TEAM][2];
    const size_t block = (size_t)p.K * p.H * p.V;
    unsigned r = blockIdx.x, k = 0;
    row_range g;
    const A* from = nullptr;
    if (r < p.nregion) {
        g = region_rows(regions, r, p.N);
        if (state) from = state + r * block;
    } else {
        const unsigned slot = r - p.nregion;
        if (!slot_segment(regions, p.nregion, p.N, cuts, slot, p.L, r, g, k)) return;
        from = carry + slot * block;
    }
    delta_lane<A, TEAM> l;
    l.place(p, blockIdx.y, p.V);
    const unsigned start = g.start + k * p.L, rows = p.L && g.end - start > p.L ? p.L : g.end - start;
    vec S[KT];
    if (g.start < g.end && l.marked(p, odd, r, blockIdx.y, p.V)) {               // (a call of no rows has no marks)
        if (k || !l.nv) return;
        load_state<A, KT>(S, from, p, l);
        delta_walk_rows<T, KT, TEAM>(p, l, Q, K, V, beta, decay, scale, g, S, O, keep);
        if (last) store_state<A, KT>(S, last + r * block, p, l);
        return;
    }
    load_state<A, KT>(S, from, p, l);
    const unsigned before = k * (p.L / DELTA_BLOCK);
    int e = 0;
    delta_walk<T, KT, TEAM, true>(p, l, lds[l.team], Q, K, V, chunks, scale, r, g.start, start, rows, S, O, keep, kept_number(g, before), false, e);
    if (last && start + rows == g.end) store_state<A, KT>(S, last + r * block, p, l);
}

constexpr int LEVEL_PLAIN = 60;                   // columns of up to this power of two, either way, are stored as they are
// What the segment in front of a slot's hands on: its state, from the region's own initial one (the first) or from zeros, and (the others) how it takes the
// state in front of it to its end: the states that the unit vectors become, times powers of two. Workgroups from `values` on along y take those. Keys of 128 columns beside values of 128: twice the
// forward pass's columns without its outputs, 278 us where that takes 249 (vector instructions 69 % of the time).
template <typename T, int KT, int TEAM>
__global__ __launch_bounds__(256, (delta_waves<typename acc_of<T>::type, KT, TEAM>())) void k_delta_local(delta_shape p, unsigned values, const uint32_t* __restrict__ regions,
                                                     const uint32_t* __restrict__ cuts, const uint32_t* __restrict__ odd, const T* __restrict__ Q, const T* __restrict__ K,
                                                     const T* __restrict__ V, const delta_chunk<typename acc_of<T>::type>* __restrict__ chunks,
                                                     const typename acc_of<T>::type* __restrict__ state, typename acc_of<T>::type* __restrict__ carry, typename acc_of<T>::type* __restrict__ through)
{
    typedef typename acc_of<T>::type A;
    typedef typename mm16<A>::vec vec;
    __shared__ typename delta_ops<T, KT>::rows lds[4 / TEAM][2];
    const unsigned slot = blockIdx.x;
    unsigned r, k;
    row_range g;
    if (!slot_segment(regions, p.nregion, p.N, cuts, slot, p.L, r, g, k)) return;
    const bool unit = blockIdx.y >= values;
    if (unit && k == 1u) return;
    delta_lane<A, TEAM> l;
    l.place(p, unit ? blockIdx.y - values : blockIdx.y, unit ? p.K : p.V);
    vec S[KT];
    const bool grows = unit && (uniform(odd[(size_t)r * p.H + l.head]) & DELTA_GROWS);
    int e = 0;
    if (unit) {
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) S[t][i] = 16u * t + l.row(i) == 16u * l.tile + l.c && l.nv ? A(1) : A(0);
    } else
        load_state<A, KT>(S, state && k == 1u ? state + (size_t)r * p.K * p.H * p.V : (const A*)nullptr, p, l);
    delta_walk<T, KT, TEAM, false>(p, l, lds[l.team], Q, K, unit ? (const T*)nullptr : V, chunks, A(1), r, g.start, g.start + (k - 1u) * p.L, p.L, S, (T*)nullptr, (A*)nullptr, 0, grows, e);
    if (unit) {
        // (powers of two only where a column's size is far from one and something grows: the carry looks at them then alone, and what only ever shrinks is not missed)
        if (grows) {
            const int size = level<A, KT>(S, e);
            if (size > -LEVEL_PLAIN && size < LEVEL_PLAIN) {
#pragma unroll
                for (int t = 0; t < KT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) S[t][i] = scaled(S[t][i], e);
                e = 0;
            }
        }
        const bool some = __any(e != 0);
        if (l.g == 0u && l.c == 0u && l.nv) through[((size_t)p.cuts * (p.K + 1u) * p.K + (size_t)slot * KT + l.tile) * p.H + l.head] = some ? A(1) : A(0);
        if (l.g == 0u && l.c < l.nv) through[((size_t)p.cuts * p.K + slot) * p.H * p.K + l.v + l.c] = (A)e;
    }
    store_state<A, KT>(S, unit ? through + slot * ((size_t)p.K * p.H * p.K) : carry + slot * ((size_t)p.K * p.H * p.V), p, l);
}

// From segment to segment: what is in front of slot k + 1 is what its own segment made of zeros and what the transition makes of what is in front of slot k; backward
// from the last segment to the first with the transposed transitions. A workgroup takes 16 columns of a head, a wave 16 rows of what comes out; what goes in lies in LDS as
// it lies in registers, and the next transition's rows come meanwhile. One step after the other: 6 us each with keys of 128 columns (67 us for
// regions of 11 segments), where a transition's 64 KB have to come, 2.4 with 64; asking for them two steps ahead gained nothing.
template <typename A, int KT>
__global__ __launch_bounds__(64 * KT) void k_delta_carry(delta_shape p, bool backward, const uint32_t* __restrict__ regions, const uint32_t* __restrict__ cuts, A* __restrict__ carry, const A* __restrict__ through)
{
    typedef typename mm16<A>::vec vec;
    __shared__ A lds[2][KT][4][64];
    const unsigned lane = threadIdx.x & 63u, t = uniform(threadIdx.x >> 6), g = lane >> 4, c = lane & 15u;
    // a workgroup per region; of many regions only those that the slots of third segments name (with two segments there is nothing to carry over one). The few workgroups that
    // have work should stand side by side in the grid where they can: those of two regions 29 slots apart took 77 us for 36.
    unsigned r = blockIdx.x, third;
    row_range rows = {0u, 0u};
    if (p.nregion > p.cuts) {
        if (!slot_segment(regions, p.nregion, p.N, cuts, blockIdx.x, p.L, r, rows, third) || third != 2u) return;
    } else
        rows = region_rows(regions, r, p.N);
    if (rows.end - rows.start <= 2u * p.L) return;
    const unsigned head = blockIdx.y / p.ns, tile = blockIdx.y % p.ns, n = (rows.end - rows.start + p.L - 1u) / p.L;      // segments: slots first + 1 .. first + n - 1
    const size_t first = rows.start / p.L, HV = (size_t)p.H * p.V, HK = (size_t)p.H * p.K, col = (size_t)head * p.V + 16u * tile + c;
    const bool here = 16u * tile + c < p.V;
    auto state = [&](size_t slot, int i) { return carry + (slot * p.K + 16u * t + mm16<A>::row(g, i)) * HV + col; };
    auto load = [&](size_t slot) {
        vec x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = here && 16u * t + mm16<A>::row(g, i) < p.K ? *state(slot, i) : A(0);
        return x;
    };
    // forward: slot i from slot i - 1 by the transition of segment i - 1, which lies in slot i; backward: slot n - i from slot n - i + 1 by that of segment n - i, in slot n - i + 1
    auto to = [&](unsigned i) { return first + (backward ? n - i : i); };
    // Where a column of a transition has an exponent, the workgroup takes one step after the other as it stands: forward what goes in is multiplied, backward what comes out.
    const A *exponents = through + (size_t)p.cuts * p.K * HK + (size_t)head * p.K, *marks = through + (size_t)p.cuts * (p.K + 1u) * HK + head;
    bool some = false;
    for (unsigned i = 2u + lane; i < n; i += 64u) some |= 16u * t < p.K && marks[((first + i) * KT + t) * p.H] != A(0);
    if (__syncthreads_or(some)) {
        vec x = load(first + (backward ? n - 1u : 1u));
#pragma unroll 1
        for (unsigned i = 2; i < n; ++i) {
            const size_t at = first + (backward ? n - i + 1u : i);
            auto grown = [&](vec v) {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = scaled(v[j], 16u * t + mm16<A>::row(g, j) < p.K ? (int)exponents[at * HK + 16u * t + mm16<A>::row(g, j)] : 0);
                return v;
            };
            if (!backward) x = grown(x);
            __syncthreads();
#pragma unroll
            for (int j = 0; j < 4; ++j) lds[0][t][j][lane] = x[j];
            __syncthreads();
            const A* m = through + at * (p.K * HK) + (size_t)head * p.K;
            x = zero16<A>();
#pragma unroll 1
            for (int s = 0; s < KT; ++s) {
                vec left, right;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const unsigned row = 16u * t + c, k = 16u * s + mm16<A>::row(g, j);
                    left[j] = row < p.K && k < p.K ? backward ? m[k * HK + row] : m[row * HK + k] : A(0);
                    right[j] = lds[0][s][j][lane];
                }
                x = product<A>(left, right, x);
            }
            x = load(to(i)) + (backward ? grown(x) : x);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (here && 16u * t + mm16<A>::row(g, j) < p.K) *state(to(i), j) = x[j];
        }
        return;
    }
    vec a[KT];
    auto transition = [&](unsigned i) {
        const A* m = through + (first + (backward ? n - i + 1u : i)) * (p.K * HK) + (size_t)head * p.K;
#pragma unroll
        for (int s = 0; s < KT; ++s)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const unsigned row = 16u * t + c, k = 16u * s + mm16<A>::row(g, j);
                a[s][j] = row < p.K && k < p.K ? backward ? m[k * HK + row] : m[row * HK + k] : A(0);
            }
    };
    const vec start = load(first + (backward ? n - 1u : 1u));
#pragma unroll
    for (int i = 0; i < 4; ++i) lds[0][t][i][lane] = start[i];
    transition(2u);
    vec own = load(to(2u));
    __syncthreads();
    for (unsigned i = 2; i < n; ++i) {
        vec x = own;
#pragma unroll
        for (int s = 0; s < KT; ++s) {
            vec b;
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = lds[i & 1u][s][j][lane];
            x = product<A>(a[s], b, x);
        }
        if (i + 1u < n) {
            transition(i + 1u);
            own = load(to(i + 1u));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            lds[~i & 1u][t][j][lane] = x[j];
            if (here && 16u * t + mm16<A>::row(g, j) < p.K) *state(to(i), j) = x[j];
        }
        __syncthreads();
    }
}

// One row of each sequence. A workgroup takes 64 columns of a head's state, a thread VEC neighbouring ones of RPT rows of it; what key and query find is added over the
// row groups in LDS. o = scale S1^T q = scale (a S0^T q + (k.q) u), so that the state is read once and written once. 128 sequences, 16 heads of 64 x 64 floats (69 MB): a call takes
// 15 us where a copy of as much takes 13.5.
template <typename T, int RPT>
__global__ __launch_bounds__(256) void k_delta_step(delta_shape p, const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V,
                                                    const typename acc_of<T>::type* __restrict__ beta, const typename acc_of<T>::type* __restrict__ decay, typename acc_of<T>::type scale,
                                                    const typename acc_of<T>::type* state, typename acc_of<T>::type* into, T* __restrict__ O)
{
    typedef typename acc_of<T>::type A;
    constexpr unsigned VEC = 4, CG = 16, RG = 16;
    __shared__ A kq[2][128], sums[3][RG][64];
    const unsigned n = blockIdx.x, parts = (p.V + 63u) / 64u, head = blockIdx.y / parts, part = blockIdx.y % parts, group = head / (p.H / p.G);
    const unsigned cg = threadIdx.x % CG, rg = threadIdx.x / CG;
    const unsigned col = part * 64u + cg * VEC, valid = col < p.V ? p.V - col : 0u;
    const size_t D = (size_t)p.H * p.V, base = (size_t)n * p.K * D + (size_t)head * p.V + col;
    const unsigned key = threadIdx.x & 127u;
    kq[threadIdx.x >> 7][key] = key < p.K ? (A)(threadIdx.x < 128u ? K[n * p.ldk + (size_t)group * p.K + key] : Q[n * p.ldq + (size_t)group * p.K + key]) : A(0);
    row_vec<A, VEC> S[RPT];
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
        const unsigned k = rg + RG * i;
        S[i].load(state + base + k * D, k < p.K ? valid : 0u);
    }
    const A a = decay ? exp(decay[n * p.ldg + head]) : A(1), b = beta[n * p.ldb + head];
    __syncthreads();
    A w[VEC], z[VEC], both = A(0);
#pragma unroll
    for (int j = 0; j < (int)VEC; ++j) w[j] = z[j] = A(0);
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
        const A k = kq[0][rg + RG * i], q = kq[1][rg + RG * i];
        both = fma(k, q, both);
#pragma unroll
        for (int j = 0; j < (int)VEC; ++j) {
            S[i].v[j] *= a;
            w[j] = fma(k, S[i].v[j], w[j]);
            z[j] = fma(q, S[i].v[j], z[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < (int)VEC; ++j) {
        sums[0][rg][cg * VEC + j] = w[j];
        sums[1][rg][cg * VEC + j] = z[j];
        sums[2][rg][cg * VEC + j] = both;
    }
    __syncthreads();
    A u[VEC];
#pragma unroll
    for (int j = 0; j < (int)VEC; ++j) {
        A ws = A(0);
#pragma unroll
        for (unsigned i = 0; i < RG; ++i) ws += sums[0][i][cg * VEC + j];
        u[j] = j < (int)valid ? b * ((A)V[n * p.ldv + (size_t)head * p.V + col + j] - ws) : A(0);
    }
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
        const unsigned k = rg + RG * i;
        const A kv = kq[0][k];
#pragma unroll
        for (int j = 0; j < (int)VEC; ++j) S[i].v[j] = fma(kv, u[j], S[i].v[j]);
        if (k < p.K) S[i].store(into + base + k * D, valid);
    }
    if (rg == 0u) {
#pragma unroll
        for (int j = 0; j < (int)VEC; ++j) {
            A zs = A(0), bs = A(0);
#pragma unroll
            for (unsigned i = 0; i < RG; ++i) { zs += sums[1][i][cg * VEC + j]; bs += sums[2][i][cg * VEC + j]; }
            if (j < (int)valid) O[n * p.ldo + (size_t)head * p.V + col + j] = (T)(scale * fma(bs, u[j], zs));
        }
    }
}

constexpr size_t DELTA_WAVES = 2048, DELTA_LEAST = 256;

delta_shape delta_shape_of(const dbk_deltarule_args& a)
{
    delta_shape s = {};
    s.N = (unsigned)a.N;
    s.nregion = (unsigned)a.nregion;
    s.H = (unsigned)a.H;
    s.G = (unsigned)a.G;
    s.K = (unsigned)a.K;
    s.V = (unsigned)a.V;
    s.ns = divup(a.V, 16);
    s.slots = (unsigned)segment_slots(a.N, DELTA_BLOCK);
    // Regions are cut into as many segments as DELTA_WAVES waves take at once, a region's last one counted as a whole one: two waves per SIMD, and none left over for a second round
    // (34 segments of 16 workgroups on 256 CUs that hold two took as long as 64). Where regions alone are half as many, only those of more than twice an even share are cut: a segment's
    // rows are walked twice, and its transition costs as much again as K columns of values.
    const size_t tracks = DELTA_WAVES / (a.H * ((s.ns + 3) / 4 * 4)), even = tracks ? tracks : 1;
    size_t L = even > 2 * a.nregion ? (a.N + even - a.nregion - 1) / (even - a.nregion) : (2 * a.N + even - 1) / even;
    L = ((L > DELTA_LEAST ? L : DELTA_LEAST) + DELTA_BLOCK - 1) / DELTA_BLOCK * DELTA_BLOCK;
    s.L = L < a.N ? (unsigned)L : 0u;
    s.cuts = s.L ? (unsigned)segment_slots(a.N, s.L) : 0u;
    s.ldq = a.ldq;
    s.ldk = a.ldk;
    s.ldv = a.ldv;
    s.ldb = a.ldbeta;
    s.ldg = a.lddecay;
    s.ldo = a.ldo;
    return s;
}

static int check_delta_shape(const dbk_deltarule_args* a)
{
    DBK_CHECK(a, "ValueError: null arguments");
    DBK_ROW_DTYPE_OK(a->dtype);
    DBK_CHECK(a->H >= 1 && a->G >= 1 && a->H % a->G == 0, "ValueError: the number of heads must be divisible by the number of key heads");
    DBK_CHECK(a->K >= 1 && a->K <= DELTA_KEY, "NotImplementedError: keys of 1 to %zu columns, got %zu", DELTA_KEY, a->K);
    DBK_CHECK(a->N < (size_t(1) << 31) && a->V < (size_t(1) << 20) && a->H < (size_t(1) << 20), "ValueError: map too large (%zu rows, %zu heads of %zu columns)", a->N, a->H, a->V);
    DBK_CHECK(a->H * ((a->V + 15) / 16 + (a->K + 15) / 16) <= 65535, "ValueError: too many heads (%zu of %zu and %zu columns)", a->H, a->K, a->V);
    DBK_CHECK(a->nregion < (size_t(1) << 24), "ValueError: too many regions (%zu)", a->nregion);
    return 0;
}

int check_delta(const dbk_deltarule_args* a)
{
    if (int rc = check_delta_shape(a)) return rc;
    DBK_CHECK(!a->N || !a->V || (a->Q && a->Kk && a->Vv && a->beta), "ValueError: null matrix");
    DBK_CHECK(a->N <= 1 || (a->ldq >= a->G * a->K && a->ldk >= a->G * a->K && a->ldv >= a->H * a->V && a->ldbeta >= a->H && (!a->decay || a->lddecay >= a->H)),
              "ValueError: row strides must be at least the number of columns");
    return 0;
}

int delta_mark(hipStream_t st, const delta_shape& s, const uint32_t* regions, uint32_t* marks, uint32_t* cuts, uint32_t* odd)
{
    k_delta_mark<<<divup(s.nregion, 4), 256, 0, st>>>(s, regions, marks, cuts, odd);
    return 0;
}

void delta_carry(hipStream_t st, const dbk_deltarule_args& a, const delta_shape& s, const delta_cuts& w, bool backward)
{
    auto launch = [&](auto t) {
        typedef decltype(t) A;
        with_key_tiles(a.K, [&](auto kt) {
            k_delta_carry<A, kt.value><<<dim3(s.nregion > s.cuts ? s.cuts : s.nregion, s.H * s.ns), 64 * kt.value, 0, st>>>(s, backward, a.regions, w.marks, (A*)w.carry, (const A*)w.through);
        });
    };
    if (a.dtype == DBK_F64) launch(double());
    else launch(float());
}

void delta_prepare(hipStream_t st, const dbk_deltarule_args& a, const delta_shape& s, const uint32_t* marks, void* chunks, void* pairs, uint32_t* odd)
{
    with_row_type(a.dtype, [&](auto t) {
        typedef decltype(t) T;
        typedef typename acc_of<T>::type A;
        with_key_tiles(a.K, [&](auto kt) {
            k_delta_prepare<T, kt.value><<<dim3((unsigned)delta_blocks(s), divup(s.H, 4)), 256, 0, st>>>(s, a.regions, marks, (const T*)a.Q, (const T*)a.Kk, (const A*)a.beta, (const A*)a.decay,
                                                                                                        (delta_chunk<A>*)chunks, (delta_pairs<A>*)pairs, odd);
        });
    });
}

namespace {

// Parts of the forward pass's workspace.
struct delta_work {
    uint32_t *marks, *odd;
    char* chunks;
    delta_cuts cuts;
    size_t bytes;
};
delta_work work_in(void* work, const dbk_deltarule_args& a, const delta_shape& s)
{
    delta_work w;
    char* p = (char*)work;
    size_t at = 0;
    w.marks = (uint32_t*)p;
    at += align16(s.slots * sizeof(uint32_t));
    w.odd = (uint32_t*)(p + at);
    at += align16(delta_odd_bytes(s));
    w.chunks = p + at;
    at += delta_chunks(s) * a.H * (a.dtype == DBK_F64 ? sizeof(delta_chunk<double>) : sizeof(delta_chunk<float>));
    const size_t A = acc_size(a.dtype);
    at = align16(at);
    w.cuts.marks = (uint32_t*)(p + at);
    at += align16(s.cuts * sizeof(uint32_t));
    w.cuts.carry = p + at;
    at += align16((size_t)s.cuts * s.K * s.H * s.V * A);
    w.cuts.through = a.keep ? (char*)a.keep + delta_kept(s) * A : p + at;
    at += delta_through(s) * A;
    w.bytes = at;
    return w;
}

}  // namespace
}  // namespace dbk

using namespace dbk;

extern "C" {

int dbk_deltarule_args_size(void) { return (int)sizeof(dbk_deltarule_args); }

int dbk_deltarule_workspace(const dbk_deltarule_args* a, int backward, size_t* work_bytes)
{
    if (int rc = check_delta(a)) return rc;
    DBK_CHECK(work_bytes, "ValueError: null result");
    *work_bytes = 0;
    if (a->N && a->V && a->nregion) *work_bytes = backward ? delta_bprop_bytes(*a) : work_in(nullptr, *a, delta_shape_of(*a)).bytes;
    clear_error();
    return 0;
}

int dbk_deltarule_kept(const dbk_deltarule_args* a, size_t* values)
{
    if (int rc = check_delta_shape(a)) return rc;
    DBK_CHECK(values, "ValueError: null result");
    // (as many segments as any number of regions may be cut into)
    dbk_deltarule_args any = *a;
    any.nregion = 0;
    const delta_shape s = a->V ? delta_shape_of(any) : delta_shape();
    *values = delta_kept(s) + delta_through(s);
    clear_error();
    return 0;
}

int dbk_deltarule(dbk_stream_t stream, const dbk_deltarule_args* a, void* work, size_t work_bytes)
{
    if (int rc = check_delta(a)) return rc;
    DBK_CHECK(!a->nregion || a->regions, "ValueError: null regions");
    DBK_CHECK(!a->N || !a->V || a->O, "ValueError: null matrix");
    DBK_CHECK(a->N <= 1 || a->ldo >= a->H * a->V, "ValueError: row strides must be at least the number of columns");
    DBK_CHECK(!a->keep || !a->state, "ValueError: states are kept for the backward pass of whole sequences, which starts from zeros: no initial state");
    if (!a->V || !a->nregion) { clear_error(); return 0; }
    const delta_shape s = delta_shape_of(*a);
    const delta_work w = work_in(work, *a, s);
    DBK_CHECK(!a->N || (work && work_bytes >= w.bytes), "ValueError: the workspace has %zu bytes, %zu are needed", work_bytes, w.bytes);
    DBK_CHECK(grid_fits(delta_blocks(s), 256), "ValueError: map too large (%zu rows, %zu regions)", a->N, a->nregion);
    hipStream_t st = as_stream(stream);
    if (a->N) {
        delta_mark(st, s, a->regions, w.marks, w.cuts.marks, w.odd);
        delta_prepare(st, *a, s, w.marks, w.chunks, nullptr, w.odd);
    }
    with_row_type(a->dtype, [&](auto t) {
        typedef decltype(t) T;
        typedef typename acc_of<T>::type A;
        with_team(a->K, s.ns, [&](auto kt, auto team) {
            if (s.L) {
                const unsigned values = team_blocks(s, team.value, s.V);
                k_delta_local<T, kt.value, team.value><<<dim3(s.cuts, values + team_blocks(s, team.value, s.K)), 256, 0, st>>>(
                    s, values, a->regions, w.cuts.marks, w.odd, (const T*)a->Q, (const T*)a->Kk, (const T*)a->Vv, (const delta_chunk<A>*)w.chunks, (const A*)a->state, (A*)w.cuts.carry,
                    (A*)w.cuts.through);
                delta_carry(st, *a, s, w.cuts, false);
            }
            k_delta_fprop<T, kt.value, team.value><<<dim3(s.nregion + s.cuts, team_blocks(s, team.value, s.V)), 256, 0, st>>>(
                s, a->regions, w.cuts.marks, w.odd, (const T*)a->Q, (const T*)a->Kk, (const T*)a->Vv, (const A*)a->beta, (const A*)a->decay, (const delta_chunk<A>*)w.chunks, (A)a->scale,
                (const A*)a->state, (const A*)w.cuts.carry, (T*)a->O,
                (A*)a->last, (A*)a->keep);
        });
    });
    DBK_LAUNCH_OK();
}

int dbk_deltarule_step(dbk_stream_t stream, const dbk_deltarule_args* a)
{
    if (int rc = check_delta(a)) return rc;
    DBK_CHECK(!a->N || !a->V || (a->O && a->state && a->last), "ValueError: null matrix or state");
    DBK_CHECK(a->N <= 1 || a->ldo >= a->H * a->V, "ValueError: row strides must be at least the number of columns");
    DBK_CHECK(grid_fits(a->N, 256, a->H * ((a->V + 63) / 64)), "ValueError: too many sequences (%zu)", a->N);
    if (!a->N || !a->V) { clear_error(); return 0; }
    const delta_shape s = delta_shape_of(*a);
    hipStream_t st = as_stream(stream);
    with_row_type(a->dtype, [&](auto t) {
        typedef decltype(t) T;
        typedef typename acc_of<T>::type A;
        with_key_tiles(a->K, [&](auto kt) {
            k_delta_step<T, kt.value><<<dim3(s.N, s.H * divup(a->V, 64)), 256, 0, st>>>(s, (const T*)a->Q, (const T*)a->Kk, (const T*)a->Vv, (const A*)a->beta, (const A*)a->decay, (A)a->scale,
                                                                                       (const A*)a->state, (A*)a->last, (T*)a->O);
        });
    });
    DBK_LAUNCH_OK();
}

}  // extern "C"
