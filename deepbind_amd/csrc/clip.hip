// The 2-norm of a set of gradients, and the gradients scaled down to a largest norm; of every model's gradients for itself where models lie side by side.
//
//   norm[b] = sqrt(sum of squares over all tensors' blocks b),  out = in * (norm[b] > max_norm ? max_norm / norm[b] : 1)
//
// Squares are formed and added in double precision, so that no float's square overflows or vanishes and a million of them lose nothing (a double's beyond 1e154 does, and counts as infinite); partial sums are added in
// a fixed order. Bound by memory: the gradients are read for the sum, read again and written. Two launches, the second of which walks the tensors from the end,
// whose values the last-level cache still holds; or one where a workgroup per model holds all of its gradients at hand (ONE_LAUNCH values). In place
// nothing is written where no norm is over the largest. 40 tensors, 92.5 million floats: 83 us for the sum (4.5 TB/s) and 137 to scale (5.4, half of what it reads from the cache).
#include "rows_common.h"

namespace dbk {

constexpr int CLIP_TENSORS = 40;                 // of a launch, whose arguments hold their table
constexpr size_t CLIP_PIECES = 4096;             // workgroups that a large set is cut into
constexpr size_t CLIP_LEAST = 4096;              // values of the smallest piece
// Values per model up to which one workgroup takes them all: sums and factors without a second launch. A call of one model's 16000 takes 13.5 us so and 18 with two launches (which is where the
// host is), of 90 models' 16000 doubles in columns 16.4 and 19.6; at 32000 those take 22.9 and 19.4, dense floats cross beyond 64000.
constexpr size_t ONE_LAUNCH = 16384;

// A tensor as its models' blocks: rows x cols of each, `next` apart.
struct clip_part {
    const void* in;
    void* out;
    size_t ldi, ldo, nexti, nexto;
    unsigned rows, cols, pieces, first;          // rows and columns of a block (a dense one: a single row), pieces of a block, number of its first piece
    size_t piece, block;                         // values of a piece (rows where there are several), values of a block
    int dtype;
};
struct clip_table {
    clip_part part[CLIP_TENSORS];
    unsigned n, all;                             // tensors of this launch, pieces of a block over all launches
    size_t nblock;
};

// f(value's place in the input, in the output) over piece `i` of a block, by the threads of a workgroup; vectors of 16 bytes where it is dense
template <typename T, int THREADS, typename F> __device__ __forceinline__ void clip_walk(const clip_part& p, const T* in, T* out, unsigned i, F f)
{
    constexpr int V = row_vec<T>::N;
    if (p.rows == 1u) {
        const size_t from = i * p.piece, to = from + p.piece < p.block ? from + p.piece : p.block;
        for (size_t e = from + threadIdx.x * V; e < to; e += THREADS * V) f(in + e, out + e, (unsigned)(to - e < (size_t)V ? to - e : V));
        return;
    }
    // rows of a wider matrix: lanes along a row, a power of two of them
    unsigned lanes = 1;
    while (lanes < THREADS && lanes * V < p.cols) lanes *= 2;
    const size_t from = i * p.piece, to = from + p.piece < p.rows ? from + p.piece : p.rows;
    for (size_t r = from + threadIdx.x / lanes; r < to; r += THREADS / lanes)
        for (unsigned c = threadIdx.x % lanes * V; c < p.cols; c += lanes * V) f(in + r * p.ldi + c, out + r * p.ldo + c, min(p.cols - c, (unsigned)V));
}

template <int THREADS> __device__ __forceinline__ double clip_sum(double v, double* lds)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) v += lds[w];
    return v;
}

template <typename F> __device__ __forceinline__ void with_clip_type(int dtype, F f)
{
    if (dtype == DBK_F32) f(float());
    else if (dtype == DBK_F64) f(double());
    else f(bf16_t());
}

template <int THREADS> __device__ __forceinline__ double clip_squares(const clip_part& p, size_t block, unsigned piece)
{
    double s = 0;
    with_clip_type(p.dtype, [&](auto t) {
        typedef decltype(t) T;
        const T* in = (const T*)p.in + block * p.nexti;
        clip_walk<T, THREADS>(p, in, (T*)nullptr, piece, [&](const T* x, T*, unsigned valid) {
            row_vec<T> v;
            v.load(x, valid);
#pragma unroll
            for (int j = 0; j < row_vec<T>::N; ++j) s = fma((double)v.v[j], (double)v.v[j], s);
        });
    });
    return s;
}

__device__ __forceinline__ double clip_factor(double norm, double most) { return norm > most ? most / norm : 1.0; }

// A factor below the type's smallest normal number has lost its digits, or is nothing, where what it makes of large gradients is neither: there floats are multiplied in double
// precision, and doubles by the two parts of the factor one after the other.
template <int THREADS> __device__ __forceinline__ void clip_scale(const clip_part& p, size_t block, unsigned piece, double norm, double most)
{
    const double factor = clip_factor(norm, most);
    if (factor == 1.0 && p.in == p.out) return;
    with_clip_type(p.dtype, [&](auto t) {
        typedef decltype(t) T;
        typedef typename acc_of<T>::type A;
        auto walk = [&](auto scaled) {
            clip_walk<T, THREADS>(p, (const T*)p.in + block * p.nexti, (T*)p.out + block * p.nexto, piece, [&](const T* x, T* y, unsigned valid) {
                row_vec<T> v;
                v.load(x, valid);
#pragma unroll
                for (int j = 0; j < row_vec<T>::N; ++j) v.v[j] = scaled(v.v[j]);
                v.store(y, valid);
            });
        };
        const A by = (A)factor;
        if (factor >= (sizeof(A) == 4 ? 0x1p-126 : 0x1p-1022)) walk([&](A v) { return v * by; });
        else if constexpr (sizeof(A) == 4) walk([&](A v) { return (A)((double)v * factor); });
        else walk([&](A v) { return v / norm * most; });
    });
}

// the tensor and piece of a workgroup, whose number counts the pieces of this launch's tensors
__device__ __forceinline__ const clip_part& clip_find(const clip_table& t, unsigned index, unsigned& piece)
{
    unsigned i = 0;
    while (i + 1u < t.n && index >= t.part[i + 1].first - t.part[0].first) ++i;
    piece = index - (t.part[i].first - t.part[0].first);
    return t.part[i];
}

__global__ __launch_bounds__(256) void k_clip_squares(clip_table t, double* __restrict__ sums)
{
    __shared__ double lds[4];
    unsigned piece;
    const clip_part& p = clip_find(t, blockIdx.x, piece);
    const double s = clip_sum<256>(clip_squares<256>(p, blockIdx.y, piece), lds);
    if (threadIdx.x == 0) sums[(size_t)blockIdx.y * t.all + p.first + piece] = s;
}

__global__ __launch_bounds__(256) void k_clip_scale(clip_table t, const double* __restrict__ sums, double most, double* __restrict__ norms)
{
    __shared__ double lds[4];
    const size_t block = gridDim.y - 1u - blockIdx.y;
    unsigned piece;
    const clip_part& p = clip_find(t, gridDim.x - 1u - blockIdx.x, piece);
    double s = 0;
    for (unsigned i = threadIdx.x; i < t.all; i += 256u) s += sums[block * t.all + i];
    const double norm = sqrt(clip_sum<256>(s, lds));
    if (p.first + piece == 0u && threadIdx.x == 0) norms[block] = norm;
    clip_scale<256>(p, block, piece, norm, most);
}

// Everything of a model in one workgroup.
__global__ __launch_bounds__(1024) void k_clip_one(clip_table t, double most, double* __restrict__ norms)
{
    __shared__ double lds[16];
    double s = 0;
    for (unsigned i = 0; i < t.n; ++i) s += clip_squares<1024>(t.part[i], blockIdx.x, 0u);
    const double norm = sqrt(clip_sum<1024>(s, lds));
    if (threadIdx.x == 0) norms[blockIdx.x] = norm;
    for (unsigned i = 0; i < t.n; ++i) clip_scale<1024>(t.part[i], blockIdx.x, 0u, norm, most);
}

namespace {

struct clip_plan {
    size_t values, most, piece, pieces;          // over all tensors' blocks; of the largest; of a piece; all pieces of a block
    bool one;
};

size_t block_values(const dbk_clip_tensor& t, size_t nblock) { return t.rows * t.cols / nblock; }
bool dense_block(const dbk_clip_tensor& t, size_t nblock)
{
    const size_t rows = t.by_rows ? t.rows / nblock : t.rows, cols = t.by_rows ? t.cols : t.cols / nblock;
    return rows <= 1 || (cols == t.ld_in && cols == t.ld_out);
}
size_t block_rows(const dbk_clip_tensor& t, size_t nblock) { return t.by_rows ? t.rows / nblock : t.rows; }
// rows of a piece where a block's rows lie apart
size_t piece_rows(const dbk_clip_tensor& t, size_t nblock, size_t piece)
{
    const size_t cols = t.by_rows ? t.cols : t.cols / nblock;
    return cols >= piece ? 1 : piece / cols;
}
size_t pieces_of(const dbk_clip_tensor& t, size_t nblock, size_t piece)
{
    const size_t v = block_values(t, nblock);
    if (!v) return 0;
    if (dense_block(t, nblock)) return (v + piece - 1) / piece;
    const size_t r = piece_rows(t, nblock, piece);
    return (block_rows(t, nblock) + r - 1) / r;
}

clip_plan plan_clip(size_t n, const dbk_clip_tensor* t, size_t nblock)
{
    clip_plan p = {};
    size_t filled = 0;
    for (size_t i = 0; i < n; ++i) { const size_t v = block_values(t[i], nblock); p.values += v; filled += v != 0; }
    // (one launch is also what an empty set takes: its norms are zeros)
    p.one = p.values <= ONE_LAUNCH && filled <= (size_t)CLIP_TENSORS;
    p.piece = (p.values * nblock + CLIP_PIECES - 1) / CLIP_PIECES;
    if (p.piece < CLIP_LEAST) p.piece = CLIP_LEAST;
    p.piece = (p.piece + 4095) / 4096 * 4096;
    if (p.one) p.piece = size_t(1) << 30;
    for (size_t i = 0; i < n; ++i) p.pieces += pieces_of(t[i], nblock, p.piece);
    return p;
}

int check_clip(size_t n, const dbk_clip_tensor* t, size_t nblock)
{
    DBK_CHECK(!n || t, "ValueError: null list of tensors");
    DBK_CHECK(nblock >= 1 && nblock <= 65535, "ValueError: 1 to 65535 blocks, got %zu", nblock);
    size_t all = 0;
    for (size_t i = 0; i < n; ++i) {
        DBK_ROW_DTYPE_OK(t[i].dtype);
        DBK_CHECK((t[i].by_rows ? t[i].rows : t[i].cols) % nblock == 0, "ValueError: tensor %zu (%zu x %zu) does not divide into %zu blocks", i, t[i].rows, t[i].cols, nblock);
        if (!t[i].rows || !t[i].cols) continue;
        DBK_CHECK(t[i].in && t[i].out, "ValueError: null tensor");
        DBK_CHECK(t[i].rows == 1 || (t[i].ld_in >= t[i].cols && t[i].ld_out >= t[i].cols), "ValueError: row strides must be at least the number of columns");
        DBK_CHECK(t[i].rows < (size_t(1) << 32) && t[i].cols < (size_t(1) << 40) / t[i].rows, "ValueError: tensor too large (%zu x %zu)", t[i].rows, t[i].cols);
        // (rows that lie apart are walked with 32-bit columns)
        DBK_CHECK(dense_block(t[i], nblock) || t[i].cols < (size_t(1) << 31), "ValueError: tensor too large (%zu x %zu)", t[i].rows, t[i].cols);
        all += t[i].rows * t[i].cols;
    }
    DBK_CHECK(all < (size_t(1) << 42), "ValueError: too many values (%zu)", all);
    return 0;
}

}  // namespace
}  // namespace dbk

using namespace dbk;

extern "C" {

int dbk_clip_gradients_workspace(size_t ntensor, const dbk_clip_tensor* tensors, size_t nblock, size_t* work_bytes)
{
    if (int rc = check_clip(ntensor, tensors, nblock)) return rc;
    DBK_CHECK(work_bytes, "ValueError: null result");
    const clip_plan p = plan_clip(ntensor, tensors, nblock);
    *work_bytes = p.one ? 0 : p.pieces * nblock * sizeof(double);
    clear_error();
    return 0;
}

int dbk_clip_gradients(dbk_stream_t stream, size_t ntensor, const dbk_clip_tensor* tensors, size_t nblock, double max_norm, double* norms, void* work, size_t work_bytes)
{
    if (int rc = check_clip(ntensor, tensors, nblock)) return rc;
    DBK_CHECK(norms, "ValueError: null norms");
    DBK_CHECK(max_norm > 0, "ValueError: the largest norm must be positive, got %g", max_norm);
    const clip_plan plan = plan_clip(ntensor, tensors, nblock);
    const size_t need = plan.one ? 0 : plan.pieces * nblock * sizeof(double);
    DBK_CHECK(!need || (work && work_bytes >= need), "ValueError: the workspace has %zu bytes, %zu are needed", work_bytes, need);
    DBK_CHECK(plan.pieces < (size_t(1) << 24), "ValueError: too many tensors (%zu)", ntensor);
    hipStream_t st = as_stream(stream);
    // the sums of all tensors before the first is scaled
    for (int pass = 0; pass < (plan.one ? 1 : 2); ++pass) {
        clip_table t = {};
        t.nblock = nblock;
        t.all = (unsigned)plan.pieces;
        unsigned first = 0, pieces = 0;
        auto launch = [&]() {
            if (plan.one) k_clip_one<<<(unsigned)nblock, 1024, 0, st>>>(t, max_norm, norms);
            else if (pass == 0) k_clip_squares<<<dim3(pieces, (unsigned)nblock), 256, 0, st>>>(t, (double*)work);
            else k_clip_scale<<<dim3(pieces, (unsigned)nblock), 256, 0, st>>>(t, (const double*)work, max_norm, norms);
            t.n = 0;
            pieces = 0;
        };
        for (size_t i = 0; i < ntensor; ++i) {
            const dbk_clip_tensor& d = tensors[i];
            const unsigned n = (unsigned)pieces_of(d, nblock, plan.piece);
            if (!n) continue;
            clip_part& p = t.part[t.n++];
            const bool dense = dense_block(d, nblock);
            const size_t rows = block_rows(d, nblock), cols = d.by_rows ? d.cols : d.cols / nblock;
            p.in = d.in;
            p.out = d.out;
            p.ldi = d.ld_in;
            p.ldo = d.ld_out;
            p.nexti = d.by_rows ? rows * d.ld_in : cols;
            p.nexto = d.by_rows ? rows * d.ld_out : cols;
            p.rows = dense ? 1u : (unsigned)rows;
            p.cols = dense ? 0u : (unsigned)cols;
            p.block = rows * cols;
            p.piece = dense ? plan.piece : piece_rows(d, nblock, plan.piece);
            p.pieces = n;
            p.first = first;
            p.dtype = d.dtype;
            first += n;
            pieces += n;
            if (t.n == (unsigned)CLIP_TENSORS && !plan.one) launch();
        }
        if (t.n || plan.one) launch();
    }
    DBK_LAUNCH_OK();
}

}  // extern "C"
