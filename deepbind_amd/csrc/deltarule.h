// The gated delta rule along the rows of every region: what its forward and backward kernels share.
//
// A head's state S (K x V) decays, is corrected by what a row's key finds in it, and is read by the row's query:
//
//   S' = a[t] S[t-1],  u[t] = b[t] (v[t] - S'^T k[t]),  S[t] = S' + k[t] u[t]^T,  o[t] = scale S[t]^T q[t],  a = exp(decay)
//
// Sixteen rows (a chunk) at once, from the state S0 before them: with the decays between rows D[i][j] = a[j+1] ... a[i], from the state to a row
// first[i] = a[0] ... a[i] and from a row to the chunk's end last[j] = a[j+1] ... a[15],
//
//   N[i][j] = D[i][j] k[i].k[j] (j < i),  P[i][j] = D[i][j] q[i].k[j] (j <= i),  T = (I + diag(b) N)^-1
//   X = V - first (K S0),  U = T (b X),  O = scale (first (Q S0) + P U),  S1 = first[15] S0 + K^T (last U)
//
// so that a chunk is a handful of 16-row products for the matrix cores. They run in the accumulation type (v_mfma_f32_16x16x4_f32, v_mfma_f64_16x16x4_f64), or on exact pieces of it
// (delta_ops): every product and sum is as exact as the states, also where rows are bfloat16. Decays are products of the rows' own factors, never quotients
// or exponentials of differences of sums, so that a factor of zero, or a long run of small ones, does what it does row by row.
//
// A matrix instruction's result and its right operand lie alike, but for the order in which the contraction runs: the lane that receives D[row(g, r)][c]
// (g = lane / 16, c = lane % 16, r = 0..3) is the one that supplies B[g][c] of instruction r, if contraction index g of it stands for row(g, r). So a product's
// result is the next one's right operand where it is, and, as the transposed result of the swapped product, its left one: states, U and their
// gradients never leave the registers. A wave holds 16 columns of a head's state and shares nothing with those that hold the others.
#pragma once
#include <type_traits>
#include "mfma_common.h"
#include "rows_common.h"

namespace dbk {

constexpr unsigned DELTA_CHUNK = 16;             // rows of a chunk: the matrix instructions' tile
constexpr unsigned DELTA_BLOCK = 64;             // rows of a block, for which states are kept and chunks are prepared by one wave
constexpr unsigned DELTA_CHUNKS = DELTA_BLOCK / DELTA_CHUNK;
constexpr size_t DELTA_KEY = 128;                // the most columns of a key

// marks of a head in a region: a chunk whose matrices leave the type's range; a row that may lengthen a state
constexpr unsigned DELTA_ODD = 1, DELTA_GROWS = 2;

struct delta_shape {
    unsigned N, nregion, H, G, K, V, ns;         // rows, regions, heads, key heads, columns of a key and of a value, tiles of 16 value columns per head
    unsigned slots;                              // blocks that are not a region's first (segment_slots)
    unsigned L, cuts;                            // rows of a segment (0: no region is cut), segments that are not a region's first
    size_t ldq, ldk, ldv, ldb, ldg, ldo;
};

template <typename A> struct mm16;
template <> struct mm16<float> {
    typedef float vec __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ vec mac(float a, float b, vec c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ unsigned row(unsigned g, unsigned r) { return 4u * g + r; }
};
template <> struct mm16<double> {
    typedef double vec __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ vec mac(double a, double b, vec c) { return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ unsigned row(unsigned g, unsigned r) { return g + 4u * r; }
};

// One 16 x 16 x 16 product: c + a b
template <typename A> __device__ __forceinline__ typename mm16<A>::vec product(typename mm16<A>::vec a, typename mm16<A>::vec b, typename mm16<A>::vec c)
{
#pragma unroll
    for (int r = 0; r < 4; ++r) c = mm16<A>::mac(a[r], b[r], c);
    return c;
}
// Two of them with the same right operand side by side, and one right operand with the left ones of many tiles: a matrix instruction waits for the one whose result it adds
// to, not for others.
template <typename A> __device__ __forceinline__ void products(typename mm16<A>::vec a, typename mm16<A>::vec b, typename mm16<A>::vec right, typename mm16<A>::vec& x, typename mm16<A>::vec& y)
{
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        x = mm16<A>::mac(a[r], right[r], x);
        y = mm16<A>::mac(b[r], right[r], y);
    }
}
template <typename A> __device__ __forceinline__ typename mm16<A>::vec zero16() { return typename mm16<A>::vec{A(0), A(0), A(0), A(0)}; }

template <typename V> __device__ __forceinline__ bool all_finite(V v)
{
    typedef decltype(v[0] * v[0]) A;
    const A z = (v[0] * A(0) + v[1] * A(0)) + (v[2] * A(0) + v[3] * A(0));
    return z == A(0);
}

// c + a b where a is a triangle, zero above the diagonal (LOWER) or below it: a row of the result takes rows of b up to itself, or from itself on. A
// product with the zeros would carry an infinity or NaN of the other rows to it as well, so where any shows the rows are done again one by one,
// with the others left out.
template <typename A, bool LOWER> __device__ __forceinline__ typename mm16<A>::vec triangle(typename mm16<A>::vec a, typename mm16<A>::vec b, typename mm16<A>::vec c, unsigned g)
{
    typename mm16<A>::vec o = product<A>(a, b, c);
    if (__any(!all_finite(o))) {
#pragma unroll 1
        for (unsigned i = 0; i < 16u; ++i) {
            typename mm16<A>::vec m;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const unsigned row = mm16<A>::row(g, r);
                m[r] = (LOWER ? row <= i : row >= i) ? b[r] : A(0);
            }
            m = product<A>(a, m, c);
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = mm16<A>::row(g, r) == i ? m[r] : o[r];
        }
    }
    return o;
}

// What one wave prepares for a chunk of a head: T and P, and per row what it decays and corrects by. Rows behind a region's last: T is the identity there, N, P and b are
// zero, and nothing decays. T is a lower triangle with ones on the diagonal and P one with its own, so that in memory they share a square, and N and D another:
// [c][row] is P[row][c] from the diagonal on and T[c][row] before it; N[row][c] and D[c][row]. (Matrices of their own are most of what 24 heads of 16 columns read and write.)
template <typename A> struct delta_chunk {
    A TP[256];
    A first[16], last[16], b[16], spare[16];
};
// and what the backward pass needs beside it
template <typename A> struct delta_pairs {
    A ND[256];
};
// A chunk's as it lies in LDS, by columns: [c][row]
template <typename A> struct delta_matrices {
    A T[256], P[256];
    A first[16], last[16], b[16], spare[16];
};

// What a chunk's matrices may hold. Decays above zero, or keys longer than one, take them beyond the type's range in 16 rows where the rows themselves may find nothing to multiply, and
// infinity times nothing is a NaN; a product that has almost vanished and grows again has lost its digits. A head with such a chunk in a region, whose keys, factors and corrections
// are all finite, is marked (prepare); three of the largest entries multiplied, as they are in a chunk, stay within the range. It goes row by row there, as the definition has it (delta_walk_rows, k_delta_bprop_rows): slow, but as far as that goes.
template <typename A> struct delta_range;
template <> struct delta_range<float> { static constexpr double most = 0x1p36, least = 0x1p-100; };
template <> struct delta_range<double> { static constexpr double most = 0x1p300, least = 0x1p-900; };

// Blocks are numbered like segments (rows_common.h): a region's first by the region, the others by their slot behind those.
struct delta_block {
    unsigned r, k, at, slot;                     // region, block within it, first row, number
    row_range g;
    unsigned rows;                               // of this block
};
__device__ __forceinline__ bool find_block(const delta_shape& p, const uint32_t* regions, const uint32_t* marks, unsigned index, delta_block& b)
{
    b.slot = index;
    if (index < p.nregion) {
        b.r = index;
        b.k = 0;
        b.g = region_rows(regions, b.r, p.N);
    } else if (!slot_segment(regions, p.nregion, p.N, marks, index - p.nregion, DELTA_BLOCK, b.r, b.g, b.k))
        return false;
    b.at = b.g.start + b.k * DELTA_BLOCK;
    if (b.at >= b.g.end) return false;
    b.rows = min(b.g.end - b.at, DELTA_BLOCK);
    return true;
}
// A chunk's matrices: a head's lie one after the other, chunks numbered like blocks, a region's first by the region, so that short regions take no more than they have.
__host__ __device__ __forceinline__ size_t delta_chunks(const delta_shape& p) { return p.nregion + (p.N + DELTA_CHUNK - 1u) / DELTA_CHUNK; }
__device__ __forceinline__ size_t chunk_number(const delta_shape& p, unsigned r, unsigned start, unsigned chunk, unsigned head)
{
    return head * delta_chunks(p) + (chunk ? (size_t)p.nregion + start / DELTA_CHUNK + chunk : r);
}
// a block's place in `keep`, which holds no region's first block
__device__ __forceinline__ size_t kept_number(row_range g, unsigned k) { return g.start / DELTA_BLOCK + k; }

// The waves that hold tiles of 16 columns of the same head are a team: 1, 2 or 4 of a workgroup's four (a head of more than 4 tiles has several), which share the head's keys and
// queries. TEAM waves; of a workgroup, 4 / TEAM teams.
template <typename A, int TEAM, int WAVES = 4> struct delta_lane {
    unsigned g, c, head, group, v;               // v: columns of V and O in front of the wave's
    unsigned nv;                                 // its columns: 16, fewer, or none
    unsigned team, thread;                       // of the workgroup's teams; of the team's threads
    unsigned tile, unit;                         // tile of the head; head and part of it
    size_t D;                                    // columns of all heads
    // cols: of a head, in tiles of 16. A team too many does the last one's work again.
    __device__ __forceinline__ void place(const delta_shape& p, unsigned index, unsigned cols)
    {
        const unsigned wave = uniform(threadIdx.x >> 6), tiles = (cols + 15u) / 16u, parts = (tiles + TEAM - 1u) / TEAM;
        g = (threadIdx.x & 63u) >> 4;
        c = threadIdx.x & 15u;
        team = wave / TEAM;
        thread = threadIdx.x & (64u * TEAM - 1u);
        unit = min(index * (unsigned)(WAVES / TEAM) + team, p.H * parts - 1u);
        head = unit / parts;
        group = head / (p.H / p.G);
        tile = unit % parts * TEAM + wave % TEAM;
        nv = tile * 16u < cols ? min(16u, cols - tile * 16u) : 0u;
        v = head * cols + (nv ? tile * 16u : 0u);
        D = (size_t)p.H * cols;
    }
    __device__ __forceinline__ unsigned row(int r) const { return mm16<A>::row(g, r); }
    // Whether this team's head goes row by row in a region; where two teams meet at the same barriers, either's.
    __device__ __forceinline__ bool marked(const delta_shape& p, const uint32_t* odd, unsigned r, unsigned index, unsigned cols) const
    {
        const uint32_t* of = odd + (size_t)r * p.H;
        if (TEAM != 2 || WAVES == TEAM) return (uniform(of[head]) & DELTA_ODD) != 0u;
        const unsigned parts = ((cols + 15u) / 16u + TEAM - 1u) / TEAM, last = p.H * parts - 1u;
        return ((uniform(of[min(index * 2u, last) / parts]) | uniform(of[min(index * 2u + 1u, last) / parts])) & DELTA_ODD) != 0u;
    }
};
template <typename F> inline void with_key_tiles(size_t K, F f)
{
    if (K <= 16) f(std::integral_constant<int, 1>());
    else if (K <= 32) f(std::integral_constant<int, 2>());
    else if (K <= 64) f(std::integral_constant<int, 4>());
    else f(std::integral_constant<int, 8>());
}

// Keys of more than 32 columns fill the LDS: there a team is always the whole workgroup, also where some of its waves have no tile and only help to fetch.
inline int team_of(size_t K, size_t tiles) { return K > 32 || tiles > 2 ? 4 : (int)tiles; }
inline unsigned team_blocks(const delta_shape& p, size_t team, size_t cols, size_t waves = 4) { return divup((size_t)p.H * (((cols + 15) / 16 + team - 1) / team), waves / team); }
template <typename F> inline void with_team(size_t K, size_t tiles, F f)
{
    auto pass = [&](auto kt) {
        if constexpr (kt.value <= 2) {
            if (tiles == 1) return f(kt, std::integral_constant<int, 1>());
            if (tiles == 2) return f(kt, std::integral_constant<int, 2>());
        }
        f(kt, std::integral_constant<int, 4>());
    };
    with_key_tiles(K, pass);
}

// A team's waves meet; a wave by itself, whose instructions on its share of LDS run in order, only keeps the compiler from changing it.
template <int TEAM> __device__ __forceinline__ void team_sync()
{
    if constexpr (TEAM == 1) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    } else
        __syncthreads();
}

// A team's keys, queries and matrices of one chunk in LDS, rows padded by 16 bytes: lanes read four neighbouring columns of 16 rows, or 16 neighbouring columns of
// four rows, without meeting in the banks.
template <typename A, int KT> struct delta_rows {
    A k[16][16 * KT + 4], q[16][16 * KT + 4];
    delta_matrices<A> c;
};
template <typename A, int W> __device__ __forceinline__ typename mm16<A>::vec tile_by_rows(const A (&m)[16][W], int t, unsigned g, unsigned c)
{
    typename mm16<A>::vec f;
#pragma unroll
    for (int r = 0; r < 4; ++r) f[r] = m[c][16u * t + mm16<A>::row(g, r)];
    return f;
}
template <typename A, int W> __device__ __forceinline__ typename mm16<A>::vec tile_by_columns(const A (&m)[16][W], int t, unsigned g, unsigned c)
{
    typename mm16<A>::vec f;
#pragma unroll
    for (int r = 0; r < 4; ++r) f[r] = m[mm16<A>::row(g, r)][16u * t + c];
    return f;
}

// Waves per SIMD that the walks are compiled for: their registers hold 4 values per lane of a state's every 16 rows. (Four teams of 32-column keys fill half the LDS.)
template <typename A, int KT, int TEAM> constexpr int delta_waves() { return sizeof(A) == 4 ? (KT > 4 || (KT == 2 && TEAM == 1) ? 2 : 4) : KT > 4 || (KT == 2 && TEAM == 1) ? 1 : 2; }

// What the walks along a region do with keys, queries and the state: w = k S (and z = q S), and S += m^T x for m of keys or queries.
template <typename T, int KT> struct delta_ops {
    typedef typename acc_of<T>::type A;
    typedef typename mm16<A>::vec vec;
    typedef delta_rows<A, KT> rows;
    template <bool BOTH, int W> static __device__ __forceinline__ void find(const A (&k)[16][W], const A (&q)[16][W], const vec (&S)[KT], vec& w, vec& z, unsigned g, unsigned c)
    {
#pragma unroll
        for (int i = 0; i < KT; ++i) {
            if (BOTH) products<A>(tile_by_rows(k, i, g, c), tile_by_rows(q, i, g, c), S[i], w, z);
            else (i & 1 ? z : w) = product<A>(tile_by_rows(k, i, g, c), S[i], i & 1 ? z : w);
        }
        if (!BOTH) w += z;
    }
    template <int W> static __device__ __forceinline__ void add(vec (&S)[KT], const A (&m)[16][W], vec x, unsigned g, unsigned c)
    {
        constexpr int N = KT < 4 ? KT : 4;
#pragma unroll
        for (int t = 0; t < KT; t += N) {
            vec f[N];
#pragma unroll
            for (int i = 0; i < N; ++i) f[i] = tile_by_columns(m, t + i, g, c);
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int i = 0; i < N; ++i) S[t + i] = mm16<A>::mac(f[i][r], x[r], S[t + i]);
        }
    }
};

// Rows kept in bfloat16 are matrix operands as they are; the float on the other side is the exact sum of three bfloat16 numbers (split3), so that three products on the 16 times
// faster bfloat16 instructions take the place of one in float, as exact as it: two tiles of the state at once where its rows are what is summed over, and one where the
// chunk's are. An infinite state or correction is a NaN here: its remainders are. Keys and queries stay bfloat16 in LDS, from where the transposing read takes them by columns:
// lane (g, i) names four columns of row 4 g + i / 4 and receives column i of rows 4 g to 4 g + 3.
template <int KT> struct delta_rows16 {
    __align__(16) unsigned short k[16][16 * KT + 8], q[16][16 * KT + 8];
    delta_matrices<float> c;
};
template <int KT> struct delta_ops<bf16_t, KT> {
    typedef mm16<float>::vec vec;
    typedef delta_rows16<KT> rows;
    typedef short quad __attribute__((ext_vector_type(4)));
    struct pieces { uint2 hi, mid, lo; };
    static __device__ __forceinline__ pieces split(vec x)
    {
        unsigned h[4], m[4], l[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) dbk_mfma::split3(x[r], l[r], m[r], h[r]);
        using dbk_mfma::pack_upper_halves;
        return {make_uint2(pack_upper_halves(h[0], h[1]), pack_upper_halves(h[2], h[3])), make_uint2(pack_upper_halves(m[0], m[1]), pack_upper_halves(m[2], m[3])),
                make_uint2(pack_upper_halves(l[0], l[1]), pack_upper_halves(l[2], l[3]))};
    }
    static __device__ __forceinline__ vec mac16(uint2 a, uint2 b, vec c) { return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(quad, a), __builtin_bit_cast(quad, b), c, 0, 0, 0); }
    static __device__ __forceinline__ vec mac32(uint2 a, uint2 a2, uint2 b, uint2 b2, vec c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(dbk_mfma::bf16x8_t, make_uint4(a.x, a.y, a2.x, a2.y)), __builtin_bit_cast(dbk_mfma::bf16x8_t, make_uint4(b.x, b.y, b2.x, b2.y)),
                                                       c, 0, 0, 0);
    }
    template <int W> static __device__ __forceinline__ uint2 by_rows(const unsigned short (&m)[16][W], int t, unsigned g, unsigned c)
    {
        return *reinterpret_cast<const uint2*>(&m[c][16u * t + 4u * g]);
    }
    template <int W> static __device__ __forceinline__ uint2 by_columns(const unsigned short (&m)[16][W], int t, unsigned g, unsigned c)
    {
        typedef __attribute__((address_space(3))) quad* at;
        return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((at)(const_cast<unsigned short*>(&m[4u * g + (c >> 2)][16u * t + 4u * (c & 3u)]))));
    }
    template <bool BOTH, int W> static __device__ __forceinline__ void find(const unsigned short (&k)[16][W], const unsigned short (&q)[16][W], const vec (&S)[KT], vec& w, vec& z, unsigned g, unsigned c)
    {
        if constexpr (KT == 1) {
            const pieces s = split(S[0]);
            const uint2 a = by_rows(k, 0, g, c), b = by_rows(q, 0, g, c);
            w = mac16(a, s.hi, mac16(a, s.mid, mac16(a, s.lo, w)));
            if (BOTH) z = mac16(b, s.hi, mac16(b, s.mid, mac16(b, s.lo, z)));
        } else {
            // (without queries three sums, one for each piece: a single one's products would wait for each other)
            vec low = zero16<float>(), mid = zero16<float>();
#pragma unroll
            for (int t = 0; t < KT; t += 2) {
                const pieces s = split(S[t]), r = split(S[t + 1]);
                const uint2 a = by_rows(k, t, g, c), a2 = by_rows(k, t + 1, g, c);
                if (BOTH) {
                    const uint2 b = by_rows(q, t, g, c), b2 = by_rows(q, t + 1, g, c);
                    w = mac32(a, a2, s.lo, r.lo, w);
                    z = mac32(b, b2, s.lo, r.lo, z);
                    w = mac32(a, a2, s.mid, r.mid, w);
                    z = mac32(b, b2, s.mid, r.mid, z);
                    w = mac32(a, a2, s.hi, r.hi, w);
                    z = mac32(b, b2, s.hi, r.hi, z);
                } else {
                    low = mac32(a, a2, s.lo, r.lo, low);
                    mid = mac32(a, a2, s.mid, r.mid, mid);
                    w = mac32(a, a2, s.hi, r.hi, w);
                }
            }
            if (!BOTH) w += mid + low;
        }
    }
    template <int W> static __device__ __forceinline__ void add(vec (&S)[KT], const unsigned short (&m)[16][W], vec x, unsigned g, unsigned c)
    {
        const pieces s = split(x);
        uint2 f[KT];
#pragma unroll
        for (int t = 0; t < KT; ++t) f[t] = by_columns(m, t, g, c);
#pragma unroll
        for (int t = 0; t < KT; ++t) S[t] = mac16(f[t], s.lo, S[t]);
#pragma unroll
        for (int t = 0; t < KT; ++t) S[t] = mac16(f[t], s.mid, S[t]);
#pragma unroll
        for (int t = 0; t < KT; ++t) S[t] = mac16(f[t], s.hi, S[t]);
    }
};

// One value as it lies in memory. Whatever is fetched ahead is read from an address that is there (of the same chunk's first row or column where its own is not) and made zero where it
// is used: a load behind a branch, or one whose value is converted at once, would be waited for there.
template <typename T> struct raw_one {
    typedef typename acc_of<T>::type A;
    typename std::conditional<sizeof(T) == 8, double, unsigned>::type r;
    __device__ __forceinline__ void load(const T* p)
    {
        if constexpr (sizeof(T) == 2) r = *reinterpret_cast<const unsigned short*>(p);
        else if constexpr (sizeof(T) == 4) r = *reinterpret_cast<const unsigned*>(p);
        else r = *p;
    }
    __device__ __forceinline__ A get(bool there)
    {
        asm volatile("" : "+v"(r));
        if constexpr (sizeof(T) == 2) return there ? __uint_as_float(r << 16) : A(0);
        else if constexpr (sizeof(T) == 4) return there ? __uint_as_float(r) : A(0);
        else return there ? r : A(0);
    }
};

// Their way there: a thread's vectors come while the chunk before is worked on (fetch), and are put into LDS when it is done (put). BOTH: queries too.
template <typename T, int KT, int TEAM, bool BOTH = true> struct delta_feed {
    typedef typename acc_of<T>::type A;
    static constexpr int EACH = KT >= TEAM ? KT / TEAM : 1, VECS = 64 * KT;      // vectors of 4 values: a thread's, a chunk's
    static constexpr int W = 4 / TEAM;                                           // a thread's values of the matrices' square, and of the vectors as long as there are any
    typedef typename row_vec<T, 4>::raw raw;
    raw k[EACH], q[EACH];
    A square[W], vectors[W];
    unsigned rows;
    __device__ __forceinline__ void fetch(const delta_shape& p, const T* Q, const T* K, const delta_chunk<A>& c, unsigned thread, unsigned rows_)
    {
        rows = rows_;
        const A *s = c.TP + W * thread, *v = c.first + min(W * thread, 64u - W);
#pragma unroll
        for (int j = 0; j < W; ++j) {
            square[j] = s[j];
            vectors[j] = v[j];
        }
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const unsigned v = thread + i * 64u * TEAM, row = v / (4u * KT), col = v % (4u * KT) * 4u;
            const T *ki = K + (row < rows ? row : 0u) * p.ldk, *qi = BOTH ? Q + (row < rows ? row : 0u) * p.ldq : nullptr;
            if (p.K % 4u == 0u) {
                const unsigned at = col < p.K ? col : 0u;
                k[i] = *reinterpret_cast<const raw*>(ki + at);
                if (BOTH) q[i] = *reinterpret_cast<const raw*>(qi + at);
            } else
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const unsigned at = col + j < p.K ? col + j : 0u;
                    k[i][j] = ki[at];
                    if (BOTH) q[i][j] = qi[at];
                }
        }
    }
    // what no chunk changes of its matrices in LDS
    static __device__ __forceinline__ void clear(delta_matrices<A>& to, unsigned thread)
    {
        if (thread >= 64u) return;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const unsigned c = thread / 4u, row = thread % 4u * 4u + j;
            if (row <= c) to.T[16u * c + row] = row == c ? A(1) : A(0);
            if (row < c) to.P[16u * c + row] = A(0);
        }
    }
    __device__ __forceinline__ void put_parts(delta_matrices<A>& to, unsigned thread) const
    {
#pragma unroll
        for (int j = 0; j < W; ++j) {
            const unsigned c = (W * thread + j) / 16u, row = (W * thread + j) % 16u;
            (row < c ? to.T + 16u * row + c : to.P + 16u * c + row)[0] = square[j];
        }
        if (W * thread >= 64u) return;
#pragma unroll
        for (int j = 0; j < W; ++j) to.first[W * thread + j] = vectors[j];
    }
    __device__ __forceinline__ void put(const delta_shape& p, delta_rows16<KT>& to, unsigned thread)
    {
        put_parts(to.c, thread);
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const unsigned v = thread + i * 64u * TEAM, row = v / (4u * KT), col = v % (4u * KT) * 4u;
            if (VECS < 64 * TEAM && v >= (unsigned)VECS) break;
            asm volatile("" : "+v"(k[i]));
            if (BOTH) asm volatile("" : "+v"(q[i]));
            typedef unsigned short quad __attribute__((ext_vector_type(4)));
            quad a = __builtin_bit_cast(quad, k[i]), b = BOTH ? __builtin_bit_cast(quad, q[i]) : a;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool there = row < rows && col + j < p.K;
                a[j] = there ? a[j] : (unsigned short)0;
                b[j] = there ? b[j] : (unsigned short)0;
            }
            *reinterpret_cast<quad*>(&to.k[row][col]) = a;
            if (BOTH) *reinterpret_cast<quad*>(&to.q[row][col]) = b;
        }
    }
    __device__ __forceinline__ void put(const delta_shape& p, delta_rows<A, KT>& to, unsigned thread)
    {
        put_parts(to.c, thread);
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const unsigned v = thread + i * 64u * TEAM, row = v / (4u * KT), col = v % (4u * KT) * 4u;
            if (VECS < 64 * TEAM && v >= (unsigned)VECS) break;
            if constexpr (sizeof(T) < 8) {
                asm volatile("" : "+v"(k[i]));
                if (BOTH) asm volatile("" : "+v"(q[i]));
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool there = row < rows && col + j < p.K;
                to.k[row][col + j] = there ? (A)k[i][j] : A(0);
                if (BOTH) to.q[row][col + j] = there ? (A)q[i][j] : A(0);
            }
        }
    }
};

// A wave's values of a chunk (of V or dO), a chunk ahead: [row(g, r)][c]
template <typename T> struct delta_values {
    typedef typename acc_of<T>::type A;
    raw_one<T> v[4];
    unsigned rows;
    // p: the chunk's first row, at the wave's first column
    template <typename L> __device__ __forceinline__ void fetch(const L& l, const T* p, size_t ld, unsigned rows_)
    {
        rows = rows_;
        const T* x = p + (l.c < l.nv ? l.c : 0u);
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r].load(x + (l.row(r) < rows ? l.row(r) : 0u) * ld);
    }
    template <typename L> __device__ __forceinline__ typename mm16<A>::vec get(const L& l)
    {
        typename mm16<A>::vec x;
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = v[r].get(l.row(r) < rows && l.c < l.nv);
        return x;
    }
};

// Tiles of keys and queries from memory, by rows: element [c][16 t + row(g, r)], as they lie there (fetch), and with zeros for rows and columns that do not exist (get).
template <typename T, int KT> struct delta_tiles {
    typedef typename acc_of<T>::type A;
    typename row_vec<T, 4>::raw f[KT];
    __device__ __forceinline__ void fetch(const T* p, size_t ld, unsigned rows, unsigned cols, unsigned g, unsigned c)
    {
        const T* x = p + (size_t)(c < rows ? c : 0u) * ld;
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            const unsigned at = 16u * t + 4u * g;
            if (sizeof(A) == 4 && cols % 4u == 0u) f[t] = *reinterpret_cast<const typename row_vec<T, 4>::raw*>(x + (at < cols ? at : 0u));
            else
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const unsigned i = 16u * t + mm16<A>::row(g, r);
                    f[t][r] = x[i < cols ? i : 0u];
                }
        }
    }
    __device__ __forceinline__ typename mm16<A>::vec get(int t, unsigned rows, unsigned cols, unsigned g, unsigned c)
    {
        if constexpr (sizeof(T) < 8) asm volatile("" : "+v"(f[t]));
        typename mm16<A>::vec v;
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = c < rows && 16u * t + mm16<A>::row(g, r) < cols ? (A)f[t][r] : A(0);
        return v;
    }
};
// and of a chunk's own matrices: [c][row(g, r)] (by rows), [row(g, r)][c] (by columns); vectors [row(g, r)]
template <typename A> __device__ __forceinline__ typename mm16<A>::vec matrix_by_rows(const A* m, unsigned g, unsigned c)
{
    typename mm16<A>::vec f;
#pragma unroll
    for (int r = 0; r < 4; ++r) f[r] = m[16u * mm16<A>::row(g, r) + c];
    return f;
}
template <typename A> __device__ __forceinline__ typename mm16<A>::vec matrix_by_columns(const A* m, unsigned g, unsigned c)
{
    typename mm16<A>::vec f;
#pragma unroll
    for (int r = 0; r < 4; ++r) f[r] = m[16u * c + mm16<A>::row(g, r)];
    return f;
}
template <typename A> __device__ __forceinline__ typename mm16<A>::vec by_row(const A* m, unsigned g)
{
    typename mm16<A>::vec f;
#pragma unroll
    for (int r = 0; r < 4; ++r) f[r] = m[mm16<A>::row(g, r)];
    return f;
}

// A wave's columns of states (blocks of K x (H V)): tile t holds rows 16 t + row(g, r).
template <typename A, int KT, int TEAM, int WAVES> __device__ __forceinline__ void load_state(typename mm16<A>::vec (&S)[KT], const A* p, const delta_shape& s, const delta_lane<A, TEAM, WAVES>& l)
{
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const unsigned k = 16u * t + l.row(r);
            S[t][r] = p && k < s.K && l.c < l.nv ? p[k * l.D + l.v + l.c] : A(0);
        }
}
template <typename A, int KT, int TEAM, int WAVES> __device__ __forceinline__ void store_state(const typename mm16<A>::vec (&S)[KT], A* p, const delta_shape& s, const delta_lane<A, TEAM, WAVES>& l)
{
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const unsigned k = 16u * t + l.row(r);
            if (k < s.K && l.c < l.nv) p[k * l.D + l.v + l.c] = S[t][r];
        }
}

// Columns of a state as c 2^e with c of size one, so that what becomes of them over many rows neither overflows nor vanishes: e takes what is taken out of S. Powers of two change no digit.
// Columns of zeros and with an infinity stay as they are; a NaN is no size and stays.
__device__ __forceinline__ float scaled(float x, int e) { return ldexpf(x, e); }
__device__ __forceinline__ double scaled(double x, int e) { return ldexp(x, e); }
template <typename A, int KT> __device__ __forceinline__ int level(typename mm16<A>::vec (&S)[KT], int& e)
{
    A m = A(0);
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) m = fmax(m, fabs(S[t][r]));
    m = fmax(m, __shfl_xor(m, 16));
    m = fmax(m, __shfl_xor(m, 32));
    const int x = m > A(0) && m * A(0) == A(0) ? ilogb(m) : 0;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) S[t][r] = scaled(S[t][r], -x);
    return e += x;
}

// Keys or queries of one row in the order of a state's registers, and what a state holds of them: the sum over a column's lanes.
template <typename A, int KT, typename T> __device__ __forceinline__ void row_tiles(typename mm16<A>::vec (&x)[KT], const T* row, unsigned K, unsigned g)
{
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const unsigned k = 16u * t + mm16<A>::row(g, r);
            x[t][r] = k < K ? (A)row[k] : A(0);
        }
}
template <typename A, int KT> __device__ __forceinline__ A found(const typename mm16<A>::vec (&x)[KT], const typename mm16<A>::vec (&S)[KT])
{
    A w = A(0);
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) w = fma(x[t][r], S[t][r], w);
    w += __shfl_xor(w, 16);
    return w + __shfl_xor(w, 32);
}
constexpr unsigned DELTA_ROWS_WGS = 512;         // workgroups that look for marked heads
// What a row multiplies the state by
template <typename A> __device__ __forceinline__ A row_factor(const delta_shape& p, const A* decay, size_t row, unsigned head) { return decay ? (A)exp((double)decay[row * p.ldg + head]) : A(1); }

// Defined in deltarule.hip.
delta_shape delta_shape_of(const dbk_deltarule_args& a);
int check_delta(const dbk_deltarule_args* a);
// odd: the marks of regions' heads (nregion, H), and behind them whether any is DELTA_ODD; cleared by the first and set by the second
int delta_mark(hipStream_t st, const delta_shape& s, const uint32_t* regions, uint32_t* marks, uint32_t* cuts, uint32_t* odd);
// chunks, and pairs where it is not null, of every block and head
void delta_prepare(hipStream_t st, const dbk_deltarule_args& a, const delta_shape& s, const uint32_t* marks, void* chunks, void* pairs, uint32_t* odd);
// What regions cut into segments need, in the workspace: whose segment a slot holds, and in front of every segment but a region's first the state (or its gradient) there.
// Transitions, by which a segment takes what is in front of it to its end, lie behind the kept states, or in the workspace where none are kept: (H, K, K) values for a segment, and behind those
// of all segments (H, K) exponents, kept as values are, of the powers of two by which the transitions' columns are larger (level), and behind those a mark per 16 columns that have any: a
// segment may grow or shrink a state beyond the type's range, where what is in front of it is small or nothing, or the segment behind does the opposite.
struct delta_cuts {
    uint32_t* marks;
    char* carry;
    char* through;
};
void delta_carry(hipStream_t st, const dbk_deltarule_args& a, const delta_shape& s, const delta_cuts& w, bool backward);
// values (not bytes) of the kept states, behind which the transitions lie
inline size_t delta_kept(const delta_shape& s) { return (size_t)s.slots * s.K * s.H * s.V; }
inline size_t delta_through(const delta_shape& s) { return (size_t)s.cuts * s.H * (s.K * (s.K + 1) + DELTA_KEY / 16); }
inline size_t delta_odd_bytes(const delta_shape& s) { return ((size_t)s.nregion * s.H + 1) * sizeof(uint32_t); }
inline size_t delta_blocks(const delta_shape& s) { return (size_t)s.nregion + s.slots; }
inline size_t align16(size_t n) { return (n + 15) / 16 * 16; }

// Defined in deltarule_bprop.hip.
size_t delta_bprop_bytes(const dbk_deltarule_args& a);

}  // namespace dbk
