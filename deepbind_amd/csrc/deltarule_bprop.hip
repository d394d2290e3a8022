// The gated delta rule's backward pass. Notation: deltarule.h; dX stands for the gradient of X, dO carries the output's scale.
//
// From the chunk's end to its start, with S0 and dS1 (the gradient of the state behind the chunk):
//
//   dU = P^T dO + last (K dS1),  dY = T^T dU (Y = b X),  dX = b dY = dV,  dW = -first dX (W = K S0)
//   dS0 = first[15] dS1 + K^T dW + Q^T (first dO)
//   dP = dO U^T,  dL = -dY U^T (L = diag(b) N, as U = Y - L U)
//   dQ = (first dO) S0^T + (dP D) K,  dK = dW S0^T + (last U) dS1^T + (dP D)^T Q + (M + M^T) K with M = b dL D below the diagonal
//   db = sum_v dY X + sum_j dL N
//
// A decay acts on every pair of rows around it, on what comes from S0, on what goes to S1 and on what passes: with E = dP P + b dL N, whose
// entries are the pairs' products of value and gradient,
//
//   ddecay[m] = sum_(i >= m > j) E[i][j] + sum_(i >= m) (q . (first dO S0^T) + k . (dW S0^T))[i] + sum_(j < m) (k . (last U dS1^T))[j] + first[15] <S0, dS1>
//
// Two kernels: a wave walks 16 columns of a head's dS up its region and leaves it behind every block of 64 rows; then all blocks are independent,
// each from the state that the forward pass kept before it and the gradient behind it. What is summed over a value's columns (dQ, dK, dP, dL) passes through LDS
// between the waves of a head, and through memory between the parts of 64 columns of wide values and between heads that share a key: added in a fixed order.
// 48 532 rows in 512 regions, 24 heads of 16 x 16 floats: 31 us up the regions, 264 for the blocks; 16 028 bfloat16 rows in two, 16 heads of 64 x 64 on 4 keys: 72 us (68 more for the
// segments from zeros and 37 for the carry), 345 for the blocks and 30 to add heads that share.
#include "deltarule.h"

namespace dbk {

// dS of a chunk's start from that of its end, chunk after chunk up `rows` rows from the last one down to row `stop` of them. What a chunk needs comes while the one
// behind it is worked on. dstates: where the gradients in front of the blocks' first rows go, from this piece's first block on; null: nowhere.
template <typename T, int KT, int TEAM>
__device__ __forceinline__ void delta_walk_back(const delta_shape& p, const delta_lane<typename acc_of<T>::type, TEAM>& l, typename delta_ops<T, KT>::rows* lds, size_t lddo, const T* Q,
                                                const T* K, const T* dO, const delta_chunk<typename acc_of<T>::type>* chunks, typename acc_of<T>::type scale, unsigned r, unsigned first,
                                                size_t row, unsigned rows, unsigned stop, typename mm16<typename acc_of<T>::type>::vec (&S)[KT], typename acc_of<T>::type* dstates)
{
    typedef typename acc_of<T>::type A;
    typedef typename mm16<A>::vec vec;
    if (rows <= stop) return;
    const T *q = Q + row * p.ldq + (size_t)l.group * p.K, *k = K + row * p.ldk + (size_t)l.group * p.K, *d0 = dO + row * lddo + l.v;
    delta_feed<T, KT, TEAM> feed;
    auto fetch = [&](unsigned t) {
        feed.fetch(p, q + t * p.ldq, k + t * p.ldk, chunks[chunk_number(p, r, first, (unsigned)(row - first + t) / DELTA_CHUNK, l.head)], l.thread, rows - t);
    };
    delta_values<T> values;
    const unsigned end = (rows - 1) / DELTA_CHUNK * DELTA_CHUNK;
    fetch(end);
    values.fetch(l, d0 + end * lddo, lddo, rows - end);
    feed.clear(lds[0].c, l.thread);
    feed.clear(lds[1].c, l.thread);
    feed.put(p, lds[end / DELTA_CHUNK & 1u], l.thread);
    if (end > stop) fetch(end - DELTA_CHUNK);
    team_sync<TEAM>();
    for (unsigned left = (end - stop) / DELTA_CHUNK + 1u, t = end; left > 0; --left, t -= DELTA_CHUNK) {
        const typename delta_ops<T, KT>::rows& here = lds[t / DELTA_CHUNK & 1u];
        const vec d = scale * values.get(l);
        if (left > 1u) {
            feed.put(p, lds[~(t / DELTA_CHUNK) & 1u], l.thread);
            values.fetch(l, d0 + (t - DELTA_CHUNK) * lddo, lddo, rows - t + DELTA_CHUNK);
        }
        if (left > 2u) fetch(t - 2u * DELTA_CHUNK);
        if (l.nv) {
            vec y = zero16<A>(), z = zero16<A>();
            delta_ops<T, KT>::template find<false>(here.k, here.k, S, y, z, l.g, l.c);
            const vec decayed = by_row(here.c.first, l.g);
            const A through = here.c.first[15];
            const vec du = triangle<A, false>(matrix_by_columns(here.c.P, l.g, l.c), d, by_row(here.c.last, l.g) * y, l.g);
            const vec fd = decayed * d;
#pragma unroll
            for (int i = 0; i < KT; ++i) S[i] *= through;
            delta_ops<T, KT>::add(S, here.q, fd, l.g, l.c);
            const vec dy = triangle<A, false>(matrix_by_columns(here.c.T, l.g, l.c), du, zero16<A>(), l.g);
            const vec dw = -(decayed * (by_row(here.c.b, l.g) * dy));
            delta_ops<T, KT>::add(S, here.k, dw, l.g, l.c);
            if (dstates && t % DELTA_BLOCK == 0) store_state<A, KT>(S, dstates + (size_t)(t / DELTA_BLOCK) * ((size_t)p.K * p.H * p.V), p, l);
        }
        team_sync<TEAM>();
    }
}

// Workgroups below nregion: a region, or the first segment of a cut one, down to its second block; the others: the segment of their slot, from the gradient carried to
// its end. In front of every block but a region's first the gradient is left behind.
template <typename T, int KT, int TEAM>
__global__ __launch_bounds__(256, (delta_waves<typename acc_of<T>::type, KT, TEAM>())) void k_delta_chain(delta_shape p, size_t lddo, const uint32_t* __restrict__ regions,
                                                     const uint32_t* __restrict__ cuts, const T* __restrict__ Q, const T* __restrict__ K,
                                                     const T* __restrict__ dO, const delta_chunk<typename acc_of<T>::type>* __restrict__ chunks, typename acc_of<T>::type scale,
                                                     const typename acc_of<T>::type* __restrict__ carry, typename acc_of<T>::type* __restrict__ dstates)
{
    typedef typename acc_of<T>::type A;
    typedef typename mm16<A>::vec vec;
    __shared__ typename delta_ops<T, KT>::rows lds[4 / TEAM][2];
    unsigned r = blockIdx.x, k = 0;
    row_range g;
    if (r < p.nregion) {
        g = region_rows(regions, r, p.N);
        if (g.end - g.start <= DELTA_BLOCK) return;
    } else if (!slot_segment(regions, p.nregion, p.N, cuts, r - p.nregion, p.L, r, g, k))
        return;
    delta_lane<A, TEAM> l;
    l.place(p, blockIdx.y, p.V);
    const size_t block = (size_t)p.K * p.H * p.V;
    const unsigned start = g.start + k * p.L;
    const bool more = p.L && g.end - start > p.L;
    vec S[KT];
    load_state<A, KT>(S, more ? carry + ((size_t)g.start / p.L + k + 1u) * block : (const A*)nullptr, p, l);
    const unsigned before = k * (p.L / DELTA_BLOCK);
    delta_walk_back<T, KT, TEAM>(p, l, lds[l.team], lddo, Q, K, dO, chunks, scale, r, g.start, start, more ? p.L : g.end - start, k ? 0u : DELTA_BLOCK, S, dstates + kept_number(g, before) * block);
}

// What a slot's segment makes of a gradient of zeros behind it
template <typename T, int KT, int TEAM>
__global__ __launch_bounds__(256, (delta_waves<typename acc_of<T>::type, KT, TEAM>())) void k_delta_chain_local(delta_shape p, size_t lddo, const uint32_t* __restrict__ regions,
                                                     const uint32_t* __restrict__ cuts, const T* __restrict__ Q, const T* __restrict__ K,
                                                     const T* __restrict__ dO, const delta_chunk<typename acc_of<T>::type>* __restrict__ chunks, typename acc_of<T>::type scale,
                                                     typename acc_of<T>::type* __restrict__ carry)
{
    typedef typename acc_of<T>::type A;
    typedef typename mm16<A>::vec vec;
    __shared__ typename delta_ops<T, KT>::rows lds[4 / TEAM][2];
    unsigned r, k;
    row_range g;
    if (!slot_segment(regions, p.nregion, p.N, cuts, blockIdx.x, p.L, r, g, k)) return;
    delta_lane<A, TEAM> l;
    l.place(p, blockIdx.y, p.V);
    const unsigned start = g.start + k * p.L;
    vec S[KT];
#pragma unroll
    for (int i = 0; i < KT; ++i) S[i] = zero16<A>();
    delta_walk_back<T, KT, TEAM>(p, l, lds[l.team], lddo, Q, K, dO, chunks, scale, r, g.start, start, min(g.end - start, p.L), 0u, S, (A*)nullptr);
    store_state<A, KT>(S, carry + blockIdx.x * ((size_t)p.K * p.H * p.V), p, l);
}

// sums over the 16 lanes of a row
template <typename A> __device__ __forceinline__ A lanes16_sum(A v)
{
    v += rotated<8>(v);
    v += rotated<4>(v);
    v += rotated<2>(v);
    return v + rotated<1>(v);
}

template <typename T> struct delta_grads {
    typedef typename acc_of<T>::type A;
    T *dQ, *dK, *dV;
    A *dbeta, *ddecay;
    size_t lddq, lddk, lddv, lddb, lddg;
    // where more than one unit (head and part of its value) has a share: (units of a key, N, G K) and (parts, N, H)
    A *dq, *dk, *db, *dg;
    unsigned parts;                              // of a value: as many tiles as a team has waves
};

// What the waves of a team show each other of one chunk: S0 and dS1 by rows of the state (a wave's own columns of them lie in its registers), dO, dY and U by rows of the
// chunk, the waves' shares of dP and dL and of what is one value a row.
// (A wave by itself leaves out the padding, with which only two of these workgroups fit a CU and not three.)
template <typename A, int KT, int TEAM> struct delta_back {
    static constexpr int W = 16 * TEAM + (TEAM > 1 ? 4 : 0);
    A s[16 * KT][W], d[16 * KT][W];
    A o[16][W], y[16][W], u[16][W];
    A pl[TEAM][2][16][17];
    A into[TEAM][16], out[TEAM][16], b[TEAM][16], through[TEAM][4];
    delta_rows<A, KT> rows;
};
template <typename A, int R, int W> __device__ __forceinline__ typename mm16<A>::vec rows_of_tile(const A (&m)[R][W], unsigned row, unsigned t, unsigned g)
{
    typename mm16<A>::vec f;
#pragma unroll
    for (int r = 0; r < 4; ++r) f[r] = m[row][16u * t + mm16<A>::row(g, r)];
    return f;
}

// The gradients of one block of 64 rows, from the state in front of it and the gradient of the state behind it: forward again over its chunks, whose states stay in registers, and
// back. Two kinds of work alternate: what runs over a head's keys (a wave's 16 columns of the value, the states in registers) and what runs over its value (16 columns of the
// key for a wave, the states in LDS), so that neither dQ and dK nor the states are ever added up or turned over between waves. Bound by what lies between: barriers, LDS and waits for
// both; the matrix units are busy for 25 % (heads of 16) and 36 % (of 64) of the time, vector instructions for 39 % and 34 %.
// Waves per SIMD it is compiled for, and with it how many registers a wave has. One more and one fewer, a call's backward pass of 47 303 rows in 512 regions: floats of 16 x 16 (24 heads) 448 us with
// three waves, 472 with two, 580 with four; 16 x 64 (8 heads) 536, 558, 839; 32 x 32 (16) 666 with two, 708 with one, 733 with three; 64 x 64 (8) 818, 1286, 1356. What the registers do not hold spills:
// 5 to 31 of them with keys of up to 16 columns in single precision, 32 (values of 32 columns) and 171 (wider) in double, where keys of more than 64 columns keep 1.3 KB a lane in memory.
template <typename A, int KT, int TEAM> constexpr int back_waves() { return sizeof(A) == 8 ? (KT == 1 && TEAM > 1 ? 2 : 1) : KT == 1 ? 3 : KT == 2 && TEAM == 1 ? 1 : KT <= 4 ? 2 : 1; }

template <typename T, int KT, int TEAM, int WAVES>
__global__ __launch_bounds__(64 * WAVES, (back_waves<typename acc_of<T>::type, KT, TEAM>())) void k_delta_bprop(delta_shape p, size_t lddo, const uint32_t* __restrict__ regions, const uint32_t* __restrict__ marks, const T* __restrict__ Q,
                                                     const T* __restrict__ K, const T* __restrict__ V, const T* __restrict__ dO,
                                                     const delta_chunk<typename acc_of<T>::type>* __restrict__ chunks, const delta_pairs<typename acc_of<T>::type>* __restrict__ pairs,
                                                     typename acc_of<T>::type scale, const typename acc_of<T>::type* __restrict__ keep,
                                                     const typename acc_of<T>::type* __restrict__ dstates, delta_grads<T> out)
{
    typedef typename acc_of<T>::type A;
    typedef typename mm16<A>::vec vec;
    constexpr int TW = KT > TEAM ? KT / TEAM : 1;
    extern __shared__ __align__(16) char lds_bytes[];
    delta_block bl;
    if (!find_block(p, regions, marks, blockIdx.x, bl)) return;
    delta_lane<A, TEAM, WAVES> l;
    l.place(p, blockIdx.y, p.V);
    delta_back<A, KT, TEAM>& lds = reinterpret_cast<delta_back<A, KT, TEAM>*>(lds_bytes)[l.team];
    const unsigned g = l.g, c = l.c, nchunk = (bl.rows + 15u) / 16u, slice = uniform(threadIdx.x >> 6) % TEAM, part = l.unit % out.parts;
    const size_t state = (size_t)p.K * p.H * p.V;
    const T *q0 = Q + (size_t)bl.at * p.ldq + (size_t)l.group * p.K, *k0 = K + (size_t)bl.at * p.ldk + (size_t)l.group * p.K;
    const T *v0 = V + (size_t)bl.at * p.ldv + l.v, *d0 = dO + (size_t)bl.at * lddo + l.v;
    auto number = [&](unsigned i) { return chunk_number(p, bl.r, bl.g.start, bl.k * DELTA_CHUNKS + i, l.head); };
    delta_feed<T, KT, TEAM> feed;
    auto fetch = [&](unsigned i) { feed.fetch(p, q0 + 16u * i * p.ldq, k0 + 16u * i * p.ldk, chunks[number(i)], l.thread, bl.rows - 16u * i); };
    delta_values<T> next;
    auto values = [&](const T* x, size_t ld, unsigned i) { next.fetch(l, x + 16u * i * ld, ld, bl.rows - 16u * i); };

    vec xs[DELTA_CHUNKS], us[DELTA_CHUNKS], sts[DELTA_CHUNKS][KT], dS[KT];
    fetch(0u);
    values(v0, p.ldv, 0u);
    feed.clear(lds.rows.c, l.thread);
    {
        vec S[KT];
        load_state<A, KT>(S, bl.k ? keep + kept_number(bl.g, bl.k) * state : (const A*)nullptr, p, l);
        load_state<A, KT>(dS, bl.at + bl.rows < bl.g.end ? dstates + kept_number(bl.g, bl.k + 1u) * state : (const A*)nullptr, p, l);
#pragma unroll
        for (int i = 0; i < (int)DELTA_CHUNKS; ++i) {
            if (i >= (int)nchunk) break;
            const unsigned n = min(bl.rows - 16u * i, 16u);
            if (i) team_sync<TEAM>();
            feed.put(p, lds.rows, l.thread);
            vec x = next.get(l), w = zero16<A>(), y;
            if (i + 1 < (int)nchunk) {
                fetch(i + 1u);
                values(v0, p.ldv, i + 1u);
            } else {
                if (i) fetch(i - 1u);
                values(d0, lddo, i);
            }
            team_sync<TEAM>();
            const delta_rows<A, KT>& here = lds.rows;
#pragma unroll
            for (int t = 0; t < KT; ++t) w = product<A>(tile_by_rows(here.k, t, g, c), S[t], w);
            const vec first = by_row(here.c.first, g), b = by_row(here.c.b, g);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                x[r] = l.row(r) < n ? x[r] - first[r] * w[r] : A(0);
                y[r] = b[r] * x[r];
            }
            xs[i] = x;
            us[i] = triangle<A, true>(matrix_by_rows(here.c.T, g, c), y, zero16<A>(), g);
#pragma unroll
            for (int t = 0; t < KT; ++t) sts[i][t] = S[t];
            if (i + 1 >= (int)nchunk) break;
            const A through = here.c.first[15];
            const vec sent = by_row(here.c.last, g) * us[i];
#pragma unroll
            for (int t = 0; t < KT; ++t) S[t] = product<A>(tile_by_columns(here.k, t, g, c), sent, through * S[t]);
        }
    }

#pragma unroll
    for (int i = (int)DELTA_CHUNKS - 1; i >= 0; --i) {
        if (i >= (int)nchunk) continue;
        const unsigned n = min(bl.rows - 16u * i, 16u);
        const size_t row = (size_t)bl.at + 16u * i;
        const delta_pairs<A>& pr = pairs[number(i)];
        if (i + 1 < (int)nchunk) {               // (the last chunk's rows are there)
            team_sync<TEAM>();
            feed.put(p, lds.rows, l.thread);
            if (i) fetch(i - 1u);
            team_sync<TEAM>();
        }
        const delta_rows<A, KT>& here = lds.rows;
        const vec d = scale * next.get(l);
        vec y = zero16<A>();
        if (i) values(d0, lddo, i - 1u);
        // (fetched here, used behind the next barriers)
        const vec Dr = matrix_by_columns(pr.ND, g, c), NDc = matrix_by_rows(pr.ND, g, c);            // D[c][row] (row < c); N[c][row] (row < c) and D[row][c] (row > c)
#pragma unroll
        for (int t = 0; t < KT; ++t) y = product<A>(tile_by_rows(here.k, t, g, c), dS[t], y);
        const vec first = by_row(here.c.first, g), b = by_row(here.c.b, g);
        const A first_c = here.c.first[c], b_c = here.c.b[c], last_c = here.c.last[c], through = here.c.first[15];
        const vec du = triangle<A, false>(matrix_by_columns(here.c.P, g, c), d, by_row(here.c.last, g) * y, g);
        const vec dy = triangle<A, false>(matrix_by_columns(here.c.T, g, c), du, zero16<A>(), g);
        const vec dx = b * dy, dw = -(first * dx), fd = first * d;
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (l.row(r) < n && c < l.nv) out.dV[(row + l.row(r)) * out.lddv + l.v + c] = (T)dx[r];
        const unsigned mine = 16u * slice + c;
        A passed = A(0);
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                lds.s[16u * t + l.row(r)][mine] = sts[i][t][r];
                lds.d[16u * t + l.row(r)][mine] = dS[t][r];
                passed = fma(sts[i][t][r], dS[t][r], passed);
            }
        passed = lanes16_sum(passed);
        if (c == 0u) lds.through[slice][g] = through * passed;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            lds.o[l.row(r)][mine] = d[r];
            lds.y[l.row(r)][mine] = dy[r];
            lds.u[l.row(r)][mine] = us[i][r];
            const A db = lanes16_sum(dy[r] * xs[i][r]);
            if (c == 0u) lds.b[slice][l.row(r)] = db;
        }
        if (i)
#pragma unroll
            for (int t = 0; t < KT; ++t)
                dS[t] = product<A>(tile_by_columns(here.q, t, g, c), fd, product<A>(tile_by_columns(here.k, t, g, c), dw, through * dS[t]));
        team_sync<TEAM>();

        // over the value: this wave's columns of the key
        vec qs[TW], ks[TW], into = zero16<A>(), sent = zero16<A>();
#pragma unroll
        for (int j = 0; j < TW; ++j) {
            const unsigned t = slice + (unsigned)TEAM * j;
            qs[j] = ks[j] = zero16<A>();
            if (t >= (unsigned)KT || 16u * t >= p.K) continue;
            vec e = zero16<A>(), s = zero16<A>();
#pragma unroll
            for (int x = 0; x < TEAM; ++x) {
                const vec s0 = rows_of_tile(lds.s, 16u * t + c, x, g);
                qs[j] = product<A>(first_c * tile_by_rows(lds.o, x, g, c), s0, qs[j]);
                e = product<A>(-(first_c * b_c) * tile_by_rows(lds.y, x, g, c), s0, e);
                s = product<A>(last_c * tile_by_rows(lds.u, x, g, c), rows_of_tile(lds.d, 16u * t + c, x, g), s);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const A k = here.k[l.row(r)][16u * t + c], q = here.q[l.row(r)][16u * t + c];
                into[r] = fma(q, qs[j][r], fma(k, e[r], into[r]));
                sent[r] = fma(k, s[r], sent[r]);
                ks[j][r] = e[r] + s[r];
            }
        }
        {
            const vec u = tile_by_rows(lds.u, (int)slice, g, c);
            const vec dp = product<A>(tile_by_rows(lds.o, (int)slice, g, c), u, zero16<A>()), dl = -product<A>(tile_by_rows(lds.y, (int)slice, g, c), u, zero16<A>());
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                lds.pl[slice][0][l.row(r)][c] = dp[r];
                lds.pl[slice][1][l.row(r)][c] = dl[r];
                const A in = lanes16_sum(into[r]), on = lanes16_sum(sent[r]);
                if (c == 0u) {
                    lds.into[slice][l.row(r)] = in;
                    lds.out[slice][l.row(r)] = on;
                }
            }
        }
        team_sync<TEAM>();

        // the team's sums, and what the pairs of rows add
        vec pr_ = zero16<A>(), lr = zero16<A>(), pc = zero16<A>(), lc = zero16<A>();    // dP and dL: [c][row], [row][c]
#pragma unroll
        for (int s = 0; s < TEAM; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                pr_[r] += lds.pl[s][0][c][l.row(r)];
                lr[r] += lds.pl[s][1][c][l.row(r)];
                pc[r] += lds.pl[s][0][l.row(r)][c];
                lc[r] += lds.pl[s][1][l.row(r)][c];
            }
        vec ar, ac, ms;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const unsigned j = l.row(r);
            ar[r] = j < c ? pr_[r] * Dr[r] : j == c ? pr_[r] : A(0);
            ac[r] = c < j ? pc[r] * NDc[r] : j == c ? pc[r] : A(0);
            ms[r] = j < c ? b_c * lr[r] * Dr[r] : c < j ? b[r] * lc[r] * NDc[r] : A(0);
        }
        const unsigned share = (l.head % (p.H / p.G)) * out.parts + part;
#pragma unroll
        for (int j = 0; j < TW; ++j) {
            const unsigned t = slice + (unsigned)TEAM * j;
            if (t >= (unsigned)KT || 16u * t >= p.K) continue;
            const vec kc = tile_by_columns(here.k, (int)t, g, c), qc = tile_by_columns(here.q, (int)t, g, c);
            const vec dq = triangle<A, true>(ar, kc, qs[j], g), dk = product<A>(ms, kc, triangle<A, false>(ac, qc, ks[j], g));
            const size_t col = (size_t)l.group * p.K + 16u * t + c;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (l.row(r) >= n || 16u * t + c >= p.K) continue;
                const size_t at = row + l.row(r);
                if (out.dq) {
                    const size_t in = ((size_t)share * p.N + at) * p.G * p.K + col;
                    out.dq[in] = dq[r];
                    out.dk[in] = dk[r];
                } else {
                    out.dQ[at * out.lddq + col] = (T)dq[r];
                    out.dK[at * out.lddk + col] = (T)dk[r];
                }
            }
        }
        if (slice == 0u) {
            const vec Pr = matrix_by_rows(here.c.P, g, c);
            vec e, before;
            A db = A(0), dg = A(0);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const unsigned j = l.row(r);
                const A ln = j < c ? lr[r] * NDc[r] : A(0);
                e[r] = j < c ? fma(b_c, ln, pr_[r] * Pr[r]) : A(0);      // (the diagonal has no decay between its rows)
                before[r] = j < c ? A(1) : A(0);
                db += ln;
            }
            vec upto = product<A>(e, before, zero16<A>());               // [i][m]: sum over j < m
            if (__any(!all_finite(upto)))                                // (one m after the other, without the pairs from m on, whose zeros would take a NaN from what is not finite in them)
#pragma unroll 1
                for (unsigned m = 0; m < 16u; ++m) {
                    vec some, one;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        some[r] = l.row(r) < m ? e[r] : A(0);
                        one[r] = A(1);
                    }
                    some = product<A>(some, one, zero16<A>());
#pragma unroll
                    for (int r = 0; r < 4; ++r) upto[r] = c == m ? some[r] : upto[r];
                }
#pragma unroll
            for (int r = 0; r < 4; ++r) dg += l.row(r) >= c ? upto[r] : A(0);
            db += __shfl_xor(db, 16);
            db += __shfl_xor(db, 32);
            dg += __shfl_xor(dg, 16);
            dg += __shfl_xor(dg, 32);
            A in = A(0), on = A(0);
#pragma unroll
            for (int s = 0; s < TEAM; ++s) {
                db += lds.b[s][c];
                dg += (lds.through[s][0] + lds.through[s][1]) + (lds.through[s][2] + lds.through[s][3]);
                in += lds.into[s][c];
                on += lds.out[s][c];
            }
            // rows from here on, and rows before
            in += from_after<1>(in);
            in += from_after<2>(in);
            in += from_after<4>(in);
            in += from_after<8>(in);
            on = from_before<1>(on);
            on += from_before<1>(on);
            on += from_before<2>(on);
            on += from_before<4>(on);
            on += from_before<8>(on);
            dg += in + on;
            if (g == 0u && c < n) {
                const size_t at = row + c;
                if (out.db) out.db[((size_t)part * p.N + at) * p.H + l.head] = db;
                else out.dbeta[at * out.lddb + l.head] = db;
                if (out.dg) out.dg[((size_t)part * p.N + at) * p.H + l.head] = dg;
                else if (out.ddecay) out.ddecay[at * out.lddg + l.head] = dg;
            }
        }
    }
}

// The gradients of marked heads, row by row, in the place of what the kernels above made of them: a team takes its columns of a head up a region, with the state's gradient in registers and
// the state in front of each row made again from the one that the forward call kept in front of its block of 64 rows.
template <typename A, int KT, int TEAM> struct delta_sums { A q[16 * KT][TEAM], k[16 * KT][TEAM], b[TEAM], g[TEAM][4]; };
template <typename T, int KT, int TEAM>
__global__ __launch_bounds__(64 * TEAM) void k_delta_bprop_rows(delta_shape p, unsigned units, size_t lddo, const uint32_t* __restrict__ regions, const uint32_t* __restrict__ odd,
                                                                const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V, const T* __restrict__ dO,
                                                                const typename acc_of<T>::type* __restrict__ beta, const typename acc_of<T>::type* __restrict__ decay,
                                                                typename acc_of<T>::type scale, const typename acc_of<T>::type* __restrict__ keep, delta_grads<T> out)
{
    typedef typename acc_of<T>::type A;
    typedef typename mm16<A>::vec vec;
    __shared__ delta_sums<A, KT, TEAM> lds;
    if (!uniform(odd[(size_t)p.nregion * p.H])) return;
    const unsigned slice = uniform(threadIdx.x >> 6);
    for (size_t i = blockIdx.x; i < (size_t)p.nregion * units; i += gridDim.x) {
        const unsigned r = (unsigned)(i / units);
        delta_lane<A, TEAM, TEAM> l;
        l.place(p, (unsigned)(i % units), p.V);
        if (!(uniform(odd[(size_t)r * p.H + l.head]) & DELTA_ODD)) continue;
        const row_range g = region_rows(regions, r, p.N);
        const bool here = l.c < l.nv;
        const unsigned part = l.unit % out.parts, share = (l.head % (p.H / p.G)) * out.parts + part;
        const T *q0 = Q + (size_t)l.group * p.K, *k0 = K + (size_t)l.group * p.K;
        vec dS[KT];
#pragma unroll
        for (int t = 0; t < KT; ++t) dS[t] = zero16<A>();
        A a, b, miss;
        vec S[KT], x[KT];                        // S: what a row leaves of the state in front of it; x: its key
        auto decayed = [&](size_t row) {
            a = row_factor(p, decay, row, l.head);
            b = beta[row * p.ldb + l.head];
            row_tiles<A, KT>(x, k0 + row * p.ldk, p.K, l.g);
#pragma unroll
            for (int t = 0; t < KT; ++t) S[t] *= a;
            miss = (here ? (A)V[row * p.ldv + l.v + l.c] : A(0)) - found<A, KT>(x, S);
        };
        auto corrected = [&]() {
#pragma unroll
            for (int t = 0; t < KT; ++t) S[t] += x[t] * (b * miss);
        };
        // eight rows at a time, whose first state is made once and those of its rows from there
        vec first[KT];
        size_t eighth = g.end;
#pragma unroll 1
        for (size_t row = g.end; row-- > g.start;) {
            if (row < eighth) {
                eighth = g.start + (row - g.start) / 8u * 8u;
                const unsigned block = ((unsigned)eighth - g.start) / DELTA_BLOCK;
                load_state<A, KT>(S, block ? keep + kept_number(g, block) * ((size_t)p.K * p.H * p.V) : (const A*)nullptr, p, l);
#pragma unroll 1
                for (size_t before = g.start + (size_t)block * DELTA_BLOCK; before < eighth; ++before) {
                    decayed(before);
                    corrected();
                }
#pragma unroll
                for (int t = 0; t < KT; ++t) first[t] = S[t];
            }
#pragma unroll
            for (int t = 0; t < KT; ++t) S[t] = first[t];
#pragma unroll 1
            for (size_t before = eighth;; ++before) {
                decayed(before);
                if (before == row) break;
                corrected();
            }
            const A d = here ? scale * (A)dO[row * lddo + l.v + l.c] : A(0), u = b * miss;
            {
                vec q[KT];
                row_tiles<A, KT>(q, q0 + row * p.ldq, p.K, l.g);
#pragma unroll
                for (int t = 0; t < KT; ++t) dS[t] += q[t] * d;
            }
            const A du = found<A, KT>(x, dS), dx = b * du, db = lanes16_sum(du * miss);
            A dg = A(0);
            __syncthreads();                     // (the sums of the row behind have been taken)
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const A dq = lanes16_sum(fma(x[t][j], u, S[t][j]) * d), dk = lanes16_sum(dS[t][j] * u - S[t][j] * dx), old = fma(-x[t][j], dx, dS[t][j]);
                    if (l.c == 0u) {
                        lds.q[16u * t + l.row(j)][slice] = dq;
                        lds.k[16u * t + l.row(j)][slice] = dk;
                    }
                    dg = fma(old, S[t][j], dg);
                    dS[t][j] = a * old;
                }
            dg = lanes16_sum(dg);
            if (l.c == 0u) {
                lds.b[slice] = db;
                lds.g[slice][l.g] = dg;
            }
            if (here && l.g == 0u) out.dV[row * out.lddv + l.v + l.c] = (T)dx;
            __syncthreads();
            for (unsigned k = threadIdx.x; k < p.K; k += 64u * TEAM) {
                A dq = A(0), dk = A(0);
#pragma unroll
                for (int s = 0; s < TEAM; ++s) {
                    dq += lds.q[k][s];
                    dk += lds.k[k][s];
                }
                const size_t col = (size_t)l.group * p.K + k;
                if (out.dq) {
                    const size_t in = ((size_t)share * p.N + row) * p.G * p.K + col;
                    out.dq[in] = dq;
                    out.dk[in] = dk;
                } else {
                    out.dQ[row * out.lddq + col] = (T)dq;
                    out.dK[row * out.lddk + col] = (T)dk;
                }
            }
            if (threadIdx.x == 0u) {
                A bs = A(0), gs = A(0);
#pragma unroll
                for (int s = 0; s < TEAM; ++s) {
                    bs += lds.b[s];
                    gs += (lds.g[s][0] + lds.g[s][1]) + (lds.g[s][2] + lds.g[s][3]);
                }
                if (out.db) out.db[((size_t)part * p.N + row) * p.H + l.head] = bs;
                else out.dbeta[row * out.lddb + l.head] = bs;
                if (out.dg) out.dg[((size_t)part * p.N + row) * p.H + l.head] = gs;
                else if (out.ddecay) out.ddecay[row * out.lddg + l.head] = gs;
            }
        }
    }
}

// out[row][col] = sum over shares of part[share][row][col], in order, for 16 rows of a block; four values a thread where they fit
template <typename A, typename T>
__device__ __forceinline__ void add_shares(size_t at, unsigned rows, size_t N, unsigned cols, unsigned shares, const A* part, T* out, size_t ld)
{
    const unsigned vecs = (cols + 3u) / 4u;
    for (unsigned i = threadIdx.x; i < rows * vecs; i += 256u) {
        const unsigned row = i / vecs, col = i % vecs * 4u, valid = cols - col;
        const A* p = part + (at + row) * cols + col;
        row_vec<A, 4> s;
        row_vec<T, 4> o;
        s.load(p, valid);
#pragma unroll 4
        for (unsigned u = 1; u < shares; ++u) {
            row_vec<A, 4> x;
            x.load(p + (size_t)u * N * cols, valid);
#pragma unroll
            for (int j = 0; j < 4; ++j) s.v[j] += x.v[j];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) o.v[j] = s.v[j];
        o.store(out + (at + row) * ld + col, valid);
    }
}

template <typename T>
__global__ __launch_bounds__(256) void k_delta_add(delta_shape p, const uint32_t* __restrict__ regions, const uint32_t* __restrict__ marks, delta_grads<T> out)
{
    delta_block bl;
    if (!find_block(p, regions, marks, blockIdx.x, bl)) return;
    const unsigned first = 16u * (blockIdx.y / 3u), what = blockIdx.y % 3u, rows = min(bl.rows - first, 16u);
    if (first >= bl.rows) return;
    const size_t at = (size_t)bl.at + first;
    if (what == 0u && out.dq) add_shares(at, rows, p.N, p.G * p.K, p.H / p.G * out.parts, out.dq, out.dQ, out.lddq);
    if (what == 1u && out.dq) add_shares(at, rows, p.N, p.G * p.K, p.H / p.G * out.parts, out.dk, out.dK, out.lddk);
    if (what == 2u && out.db) add_shares(at, rows, p.N, p.H, out.parts, out.db, out.dbeta, out.lddb);
    if (what == 2u && out.dg) add_shares(at, rows, p.N, p.H, out.parts, out.dg, out.ddecay, out.lddg);
}

namespace {

struct delta_bprop_work {
    uint32_t *marks, *odd;
    char *chunks, *pairs, *dstates, *dq, *dk, *db, *dg;
    unsigned parts;
    delta_cuts cuts;
    size_t bytes;
};

// Tiles of a value that a team takes at once: its states' share of the LDS, in double precision and with keys of more than 64 columns, is that of two.
unsigned back_team(const dbk_deltarule_args& a) { return a.dtype == DBK_F64 && a.K > 64 ? 2u : (unsigned)team_of(a.K, (a.V + 15) / 16); }

delta_bprop_work bprop_work_in(void* work, const dbk_deltarule_args& a, const delta_shape& s)
{
    delta_bprop_work w = {};
    char* base = (char*)work;
    size_t at = 0;
    auto take = [&](size_t n) { char* p = base + at; at += align16(n); return p; };
    const size_t A = acc_size(a.dtype), units = delta_chunks(s) * a.H;
    w.parts = (s.ns + back_team(a) - 1) / back_team(a);
    w.marks = (uint32_t*)take(s.slots * sizeof(uint32_t));
    w.odd = (uint32_t*)take(delta_odd_bytes(s));
    w.chunks = take(units * (A == 8 ? sizeof(delta_chunk<double>) : sizeof(delta_chunk<float>)));
    w.pairs = take(units * (A == 8 ? sizeof(delta_pairs<double>) : sizeof(delta_pairs<float>)));
    w.dstates = take((size_t)s.slots * a.K * a.H * a.V * A);
    const size_t shares = a.H / a.G * w.parts;
    if (shares > 1) {
        w.dq = take(shares * a.N * a.G * a.K * A);
        w.dk = take(shares * a.N * a.G * a.K * A);
    }
    if (w.parts > 1) {
        w.db = take((size_t)w.parts * a.N * a.H * A);
        w.dg = take((size_t)w.parts * a.N * a.H * A);
    }
    w.cuts.marks = (uint32_t*)take(s.cuts * sizeof(uint32_t));
    w.cuts.carry = take((size_t)s.cuts * s.K * s.H * s.V * A);
    w.cuts.through = (char*)a.keep + delta_kept(s) * A;
    w.bytes = at;
    return w;
}

}  // namespace

size_t delta_bprop_bytes(const dbk_deltarule_args& a) { return bprop_work_in(nullptr, a, delta_shape_of(a)).bytes; }

}  // namespace dbk

using namespace dbk;

extern "C" {

int dbk_deltarule_bprop(dbk_stream_t stream, const dbk_deltarule_args* a, void* work, size_t work_bytes)
{
    if (int rc = check_delta(a)) return rc;
    DBK_CHECK(!a->nregion || a->regions, "ValueError: null regions");
    DBK_CHECK(!a->N || !a->V || (a->dO && a->dQ && a->dK && a->dV && a->dbeta), "ValueError: null matrix");
    DBK_CHECK(a->decay || !a->ddecay, "ValueError: no decay, no gradient of it");
    DBK_CHECK(!a->N || !a->V || a->keep, "ValueError: the states that the forward call kept are needed");
    DBK_CHECK(a->N <= 1 || (a->lddo >= a->H * a->V && a->lddv >= a->H * a->V && a->lddq >= a->G * a->K && a->lddk >= a->G * a->K && a->lddbeta >= a->H && (!a->ddecay || a->ldddecay >= a->H)),
              "ValueError: row strides must be at least the number of columns");
    if (!a->N || !a->V || !a->nregion) { clear_error(); return 0; }
    const delta_shape s = delta_shape_of(*a);
    const delta_bprop_work w = bprop_work_in(work, *a, s);
    DBK_CHECK(work && work_bytes >= w.bytes, "ValueError: the workspace has %zu bytes, %zu are needed", work_bytes, w.bytes);
    DBK_CHECK(grid_fits(delta_blocks(s), 256), "ValueError: map too large (%zu rows, %zu regions)", a->N, a->nregion);
    hipStream_t st = as_stream(stream);
    delta_mark(st, s, a->regions, w.marks, w.cuts.marks, w.odd);
    delta_prepare(st, *a, s, w.marks, w.chunks, w.pairs, w.odd);
    int rc = 0;
    with_row_type(a->dtype, [&](auto t) {
        typedef decltype(t) T;
        typedef typename acc_of<T>::type A;
        delta_grads<T> out = {(T*)a->dQ, (T*)a->dK, (T*)a->dV, (A*)a->dbeta, (A*)a->ddecay, a->lddq, a->lddk, a->lddv, a->lddbeta, a->ldddecay,
                              (A*)w.dq, (A*)w.dk, (A*)w.db, a->ddecay ? (A*)w.dg : nullptr, w.parts};
        with_team(a->K, s.ns, [&](auto kt, auto team) {
            const unsigned columns = team_blocks(s, team.value, s.V);
            if (s.L) {
                k_delta_chain_local<T, kt.value, team.value><<<dim3(s.cuts, columns), 256, 0, st>>>(
                    s, a->lddo, a->regions, w.cuts.marks, (const T*)a->Q, (const T*)a->Kk, (const T*)a->dO, (const delta_chunk<A>*)w.chunks, (A)a->scale, (A*)w.cuts.carry);
                delta_carry(st, *a, s, w.cuts, true);
            }
            k_delta_chain<T, kt.value, team.value><<<dim3(s.nregion + s.cuts, columns), 256, 0, st>>>(
                s, a->lddo, a->regions, w.cuts.marks, (const T*)a->Q, (const T*)a->Kk, (const T*)a->dO, (const delta_chunk<A>*)w.chunks, (A)a->scale, (const A*)w.cuts.carry, (A*)w.dstates);
            constexpr bool half = sizeof(A) == 8 && kt.value == 8;
            constexpr int TEAM = half ? 2 : team.value, WAVES = half ? 2 : 4;
            constexpr size_t lds = WAVES / TEAM * sizeof(delta_back<A, kt.value, TEAM>);
            static_assert(lds <= 163840, "a workgroup's shared memory");
            auto kernel = k_delta_bprop<T, kt.value, TEAM, WAVES>;
            if (lds > 65536 && hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess) { rc = 1; return; }
            kernel<<<dim3((unsigned)delta_blocks(s), team_blocks(s, TEAM, s.V, WAVES)), 64 * WAVES, lds, st>>>(
                s, a->lddo, a->regions, w.marks, (const T*)a->Q, (const T*)a->Kk, (const T*)a->Vv, (const T*)a->dO, (const delta_chunk<A>*)w.chunks, (const delta_pairs<A>*)w.pairs,
                (A)a->scale, (const A*)a->keep, (const A*)w.dstates, out);
            const unsigned units = team_blocks(s, TEAM, s.V, TEAM);
            k_delta_bprop_rows<T, kt.value, TEAM><<<DELTA_ROWS_WGS, 64 * TEAM, 0, st>>>(s, units, a->lddo, a->regions, w.odd, (const T*)a->Q, (const T*)a->Kk, (const T*)a->Vv, (const T*)a->dO,
                                                                                        (const A*)a->beta, (const A*)a->decay, (A)a->scale, (const A*)a->keep, out);
        });
        if (!rc && (w.dq || w.db)) k_delta_add<T><<<dim3((unsigned)delta_blocks(s), 3 * DELTA_CHUNKS), 256, 0, st>>>(s, a->regions, w.marks, out);
    });
    DBK_CHECK(!rc, "RuntimeError: the device has too little shared memory for a workgroup");
    DBK_LAUNCH_OK();
}

}  // extern "C"
