// The optimiser's operators over a LIST of tensors: 2-norm and largest modulus of the whole list, scaling to a bound of one of them, momentum
// step with that scaling in its registers (include/ctm_hip.h: ctm_grad_norms, ctm_grad_clip, ctm_sgd_step).
//
//   N2 = (sum_t sum_i |x_ti|^2)^1/2,  Ninf = max |x_ti|,  c = 1 if N <= max_norm else max_norm / N,
//   clip  y = c x          step  g' = c g,  m <- mu m + (1 - tau) g'  (first step: m <- g'),  p <- p - lr m
//
// All of it is bound by memory traffic on long lists (3 ... 9 flop per 8 ... 40 bytes) and by launches on short ones.  Nothing is kept between
// calls, nothing is read back by the host, no atomics and no memset: every sum has a fixed order, and a captured call replays as it ran.
#include "ctm_common.h"
#include "grads_lists.h"

namespace {

typedef double d2 __attribute__((ext_vector_type(2)));
typedef d2 d2u __attribute__((aligned(8)));          // 16-byte access at 8-byte alignment: views into a flat buffer start anywhere

template <bool NT> __device__ __forceinline__ d2 load2(const double* x) {
    if (NT) return __builtin_nontemporal_load((const d2u*)x);
    return *(const d2u*)x;
}
template <bool NT> __device__ __forceinline__ void store2(double* x, d2 v) {
    if (NT) __builtin_nontemporal_store((d2u)v, (d2u*)x);
    else *(d2u*)x = v;
}

// The tensor that holds chunk q: each lane of a wave compares N / 64 table entries, the count of those at or below q is its number.  The tensor
// found last is tried first: chunks of long tensors need no lookup.
template <int NP> struct Finder {
    static constexpr int R = Table<NP>::N / 64;
    const Table<NP>& t;
    unsigned mine[R];
    unsigned f = 0, l = 0;             // chunks of the tensor: f ... l - 1
    long long n = 0;                   // its doubles
    double* p[NP] = {};
    __device__ __forceinline__ explicit Finder(const Table<NP>& table) : t(table) {
#pragma unroll
        for (int j = 0; j < R; ++j) mine[j] = t.first[64 * j + (threadIdx.x & 63) + 1];
    }
    __device__ __forceinline__ void find(unsigned q, int chunk) {
        if (q >= f && q < l) return;
        int k = 0;
#pragma unroll
        for (int j = 0; j < R; ++j) k += __popcll(__ballot(mine[j] <= q));
        k = __builtin_amdgcn_readfirstlane(k);
        f = t.first[k];
        l = t.first[k + 1];
        n = (long long)(l - f - 1) * chunk + t.tail[k] + 1;
#pragma unroll
        for (int j = 0; j < NP; ++j) p[j] = t.base[j][(t.which[k] >> (2 * j)) & 3] + t.offset[j][k];
    }
};

// Runs body(pointers, first double, length of the tensor) over this workgroup's chunks: every gridDim.x-th one, so that all workgroups sweep the
// list together (measured on 545 MB: 87 us for the norm pass against 95 with one contiguous share per workgroup, 185 against 223 for the
// scaling).
template <int NP, class F> __device__ __forceinline__ void chunks(const Table<NP>& t, F&& body) {
    Finder<NP> at(t);
    const unsigned G = t.first[Table<NP>::N];
    for (unsigned q = blockIdx.x; q < G; q += gridDim.x) {
        at.find(q, CHUNK);
        body(at.p, (long long)(q - at.f) * CHUNK, at.n);
    }
}

// Elements a + 2 u THREADS (+ 1) of this thread, zero behind the end of the tensor
template <bool NT> __device__ __forceinline__ void load_chunk(d2 (&v)[UNROLL], const double* x, long long a, long long n) {
    const long long i = a + 2 * threadIdx.x;
    if (a + CHUNK <= n) {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) v[u] = load2<NT>(x + i + u * 2 * THREADS);
    } else {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const long long j = i + u * 2 * THREADS;
            v[u] = d2{0.0, 0.0};
            if (j + 1 < n) v[u] = load2<NT>(x + j);
            else if (j < n) v[u].x = x[j];               // (real tensors of odd length)
        }
    }
}
template <bool NT> __device__ __forceinline__ void store_chunk(const d2 (&v)[UNROLL], double* x, long long a, long long n) {
    const long long i = a + 2 * threadIdx.x;
    if (a + CHUNK <= n) {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) store2<NT>(x + i + u * 2 * THREADS, v[u]);
    } else {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const long long j = i + u * 2 * THREADS;
            if (j + 1 < n) store2<NT>(x + j, v[u]);
            else if (j < n) x[j] = v[u].x;
        }
    }
}

// Sum of squares in three ranges (J. L. Blue, ACM TOMS 4 (1978) 15): elements between 2^-480 and 2^480 are squared as they are, the others scaled
// by 2^600 or 2^-600 first, so that neither overflow nor underflow of a square changes the norm.  The largest modulus is kept as the bit pattern
// of a non-negative double: the order of the patterns is that of the numbers, with NaN behind infinity, so a NaN survives the maximum.
struct Acc {
    double big = 0.0, med = 0.0, small = 0.0;
    unsigned long long top = 0;        // real: max |x|;  complex: max |z|^2 of the middle range
    unsigned long long top_far = 0;    // complex: max |z| of the others
};

__device__ __forceinline__ unsigned long long bits(double x) { return (unsigned long long)__double_as_longlong(x); }
__device__ __forceinline__ unsigned long long umax(unsigned long long a, unsigned long long b) { return a > b ? a : b; }
constexpr unsigned EXP_LO = 1023 - 480, EXP_SPAN = 960;
__device__ __forceinline__ bool middle(double x) { return (((unsigned)__double2hiint(x) >> 20) & 0x7ffu) - EXP_LO < EXP_SPAN; }

__device__ __forceinline__ void add_far(Acc& a, double x) {
    const unsigned e = ((unsigned)__double2hiint(x) >> 20) & 0x7ffu;
    if (e >= EXP_LO + EXP_SPAN) { const double s = x * 0x1p-600; a.big = fma(s, s, a.big); }
    else if (e >= EXP_LO) a.med = fma(x, x, a.med);
    else { const double s = x * 0x1p600; a.small = fma(s, s, a.small); }
}

template <bool CPLX> __device__ __forceinline__ void add(Acc& a, d2 v) {
    // (zeros take the short way too: the imaginary parts of real data, masked entries)
    if ((middle(v.x) || v.x == 0.0) && (middle(v.y) || v.y == 0.0)) {
        const double s = fma(v.x, v.x, v.y * v.y);
        a.med += s;
        if (CPLX) a.top = umax(a.top, bits(s));
    } else {
        add_far(a, v.x);
        add_far(a, v.y);
        // (hypot of an infinity and a NaN is infinite)
        if (CPLX) a.top_far = umax(a.top_far, bits(v.x != v.x || v.y != v.y ? __builtin_nan("") : hypot(v.x, v.y)));
    }
    if (!CPLX) { a.top = umax(a.top, bits(fabs(v.x))); a.top = umax(a.top, bits(fabs(v.y))); }
}

struct Part { double big, med, small; unsigned long long top; };

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
    return x;
}

__device__ __forceinline__ void join(Part& p, const Part& q) {
    p.big += q.big; p.med += q.med; p.small += q.small; p.top = umax(p.top, q.top);
}

// Result of a workgroup of `WAVES` waves, the same bits on all its threads.
template <int WAVES> __device__ __forceinline__ Part reduce_block(Part p) {
    __shared__ Part sh[WAVES];
    p.med = wave_sum(p.med);
    if (__any(p.big != 0.0)) p.big = wave_sum(p.big);          // (true for NaN)
    if (__any(p.small != 0.0)) p.small = wave_sum(p.small);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) p.top = umax(p.top, __shfl_xor(p.top, o));
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = p;
    __syncthreads();
    Part r = sh[0];
#pragma unroll 3                   // (not all 16 parts in registers at once, next to the list that small_kernel keeps there)
    for (int w = 1; w < WAVES; ++w) join(r, sh[w]);
    return r;
}

template <bool CPLX> __device__ __forceinline__ Part part_of(const Acc& a) {
    Part p{a.big, a.med, a.small, a.top};
    if (CPLX) p.top = umax(bits(sqrt(__longlong_as_double((long long)a.top))), a.top_far);
    return p;
}

struct Bound { double max_norm; int inf_norm; };      // max_norm < 0: no bound

// What the kernels multiply by: c itself, or, for a c below the normal range (a norm above 2^1022 times the bound), where a double has no 53 bits left
// for it, -a / n: then y = (x a / n) (max_norm / a), whose first product is at most a.  a = 4 keeps a / n normal, a = 1 the bits of a bound that
// lies at the end of the range itself.  (One double, whose sign tells which: two cost the step a wave per SIMD, 19.9 us against 19.6 on 61 MB.)
__device__ __forceinline__ double tiny_a(double max_norm) { return max_norm < 0x1p-1020 ? 1.0 : 4.0; }
__device__ __forceinline__ double multiplier(double n, double max_norm) {
    const bool tiny = max_norm < n * 0x1p-1022 && max_norm > 0.0 && n <= 0x1.fffffffffffffp1023;
    return (tiny ? -tiny_a(max_norm) : max_norm) / n;                                      // (NaN norm: NaN)
}
template <int N> __device__ __forceinline__ void scale(d2 (&v)[N], double k, double max_norm) {
    if (k < 0.0) {
        const double s = max_norm / tiny_a(max_norm);
#pragma unroll
        for (int u = 0; u < N; ++u) v[u] = v[u] * -k * s;
    } else {
#pragma unroll
        for (int u = 0; u < N; ++u) v[u] *= k;
    }
}

// N2, Ninf and the multiplier from the three range sums
struct Norms { double n2, ninf, k; };
__device__ __forceinline__ Norms finish(const Part& p, Bound bd) {
    Norms r;
    if (p.big != 0.0) r.n2 = sqrt(fma(p.med * 0x1p-600, 0x1p-600, p.big)) * 0x1p600;
    else if (p.med != 0.0) r.n2 = sqrt(fma(p.small * 0x1p-600, 0x1p-600, p.med));
    else r.n2 = sqrt(p.small) * 0x1p-600;
    r.ninf = __longlong_as_double((long long)p.top);
    const double n = bd.inf_norm ? r.ninf : r.n2;
    r.k = (bd.max_norm < 0.0 || n <= bd.max_norm) ? 1.0 : multiplier(n, bd.max_norm);
    return r;
}
__device__ __forceinline__ void put_norms(const Norms& r, Bound bd, double* ws) {
    ws[0] = r.n2;
    ws[1] = r.ninf;
    ws[2] = r.k < 0.0 ? bd.max_norm / (bd.inf_norm ? r.ninf : r.n2) : r.k;
    ws[3] = r.k;
}

// First pass: partial results of the workgroups.
template <bool CPLX, bool NT>
__global__ __launch_bounds__(THREADS) void norm_partials_kernel(const Table<1> t, Part* out) {
    Acc acc;
    chunks<1>(t, [&](double* const* p, long long a, long long n) {
        d2 v[UNROLL];
        load_chunk<NT>(v, p[0], a, n);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) add<CPLX>(acc, v[u]);
    });
    const Part p = reduce_block<THREADS / 64>(part_of<CPLX>(acc));
    if (threadIdx.x == 0) out[blockIdx.x] = p;
}

// Norms from the partial results, by a workgroup of T threads, in an order that depends on T and np alone
template <int T> __device__ __forceinline__ Norms join_partials(const Part* part, int np, Bound bd) {
    Part p{0.0, 0.0, 0.0, 0};
    for (int i = threadIdx.x; i < np; i += T) join(p, part[i]);
    return finish(reduce_block<T / 64>(p), bd);
}

__global__ __launch_bounds__(1024) void norm_finish_kernel(const Part* part, int np, Bound bd, double* ws) {
    const Norms r = join_partials<1024>(part, np, bd);
    if (threadIdx.x == 0) put_norms(r, bd, ws);
}

// Where the second pass gets its factor from.  Lists of at most LONG chunks: every workgroup joins the partial results by itself (all get the same
// bits) while its part of the list is on its way, which saves the 4 us of a kernel in between.  Longer ones, of many times more workgroups
// than partial results: from ws, where norm_finish_kernel left it (np = 0).
struct Source { const Part* part; int np; Bound bd; double* ws; bool write; };      // write: one workgroup leaves the norms in ws
__device__ __forceinline__ double factor(const Source& s) {
    if (s.bd.max_norm < 0.0) return 1.0;
    if (s.np == 0) return s.ws[3];
    const Norms r = join_partials<THREADS>(s.part, s.np, s.bd);
    if (s.write && blockIdx.x == 0 && threadIdx.x == 0) put_norms(r, s.bd, s.ws);
    return r.k;
}

// y = c x (p[0] = x, p[1] = y).  In place a list inside the bound (c = 1) is neither read nor written.
template <bool NT>
__global__ __launch_bounds__(THREADS) void clip_kernel(const Table<2> t, const Source s) {
    double k = 0.0;
    bool known = false;
    chunks<2>(t, [&](double* const* p, long long a, long long n) {
        d2 v[UNROLL];
        const bool apart = p[0] != p[1];
        if (apart) load_chunk<false>(v, p[0], a, n);
        if (!known) { k = factor(s); known = true; }
        if (!apart) {
            if (k == 1.0) return;
            load_chunk<false>(v, p[0], a, n);
        }
        scale(v, k, s.bd.max_norm);
        store_chunk<NT>(v, p[1], a, n);
    });
}

struct Step { double lr, mu, one_minus_tau; int first; };

// d = c g -> the new momentum (MOMENTUM), p -> the new parameters
template <bool MOMENTUM> __device__ __forceinline__ void step_pair(d2& p, d2& d, d2 m, const Step& s) {
    if (MOMENTUM && !s.first) d = m * s.mu + d * s.one_minus_tau;
    p -= d * s.lr;
}

// p[0] = parameters, p[1] = gradients, p[2] = momentum buffers (MOMENTUM)
template <bool MOMENTUM, bool NT>
__global__ __launch_bounds__(THREADS) void sgd_kernel(const Table<MOMENTUM ? 3 : 2> t, const Step s, const Source src) {
    double k = 0.0;
    bool known = false;
    chunks<MOMENTUM ? 3 : 2>(t, [&](double* const* p, long long a, long long n) {
        d2 x[UNROLL], d[UNROLL], m[UNROLL];
        load_chunk<false>(d, p[1], a, n);
        if (MOMENTUM && !s.first) load_chunk<false>(m, p[MOMENTUM ? 2 : 0], a, n);
        load_chunk<false>(x, p[0], a, n);
        if (!known) { k = factor(src); known = true; }
        scale(d, k, src.bd.max_norm);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) step_pair<MOMENTUM>(x[u], d[u], m[u], s);
        if (MOMENTUM) store_chunk<NT>(d, p[MOMENTUM ? 2 : 0], a, n);
        store_chunk<NT>(x, p[0], a, n);
    });
}

// Short lists: one workgroup, one launch, the list in registers between the norm and its second use.  Its 16 waves take pieces of 128 doubles,
// ROUNDS of them each: up to there one workgroup is faster than two launches of many (one tensor of n doubles, graph replays, us: norms n = 32
// 4.5 and 6.6, 12288 6.2 and 6.8, 16384 6.8 and 6.8; clipping 4.6 and 6.1, 6144 6.0 and 6.4, 8192 6.5 and 6.5; step with momentum 4.5 and 7.2,
// 6144 6.6 and 6.8, 8192 7.2 and 6.8; 32 tensors of 128: norms 5.4 and 7.1, clipping 6.3 and 7.0).
constexpr int SMALL_THREADS = 1024, SMALL_WAVES = SMALL_THREADS / 64;
enum { OP_NORMS, OP_CLIP, OP_SGD, OP_SGD_MOMENTUM };
template <int OP> struct Shape {
    static constexpr int NP = OP == OP_NORMS ? 1 : OP == OP_SGD_MOMENTUM ? 3 : 2, READ = OP >= OP_SGD ? 1 : 0, ROUNDS = OP == OP_NORMS ? 6 : 3;
};

__device__ __forceinline__ d2 load_piece(const double* x, int i, int n) {
    d2 v = {0.0, 0.0};
    if (i + 1 < n) v = load2<false>(x + i);
    else if (i < n) v.x = x[i];
    return v;
}
__device__ __forceinline__ void store_piece(d2 v, double* x, int i, int n) {
    if (i + 1 < n) store2<false>(x + i, v);
    else if (i < n) x[i] = v.x;
}

template <int OP, bool CPLX>
__global__ __launch_bounds__(SMALL_THREADS) void small_kernel(const Table<Shape<OP>::NP> t, const Bound bd, const Step s, double* ws) {
    using S = Shape<OP>;
    Finder<S::NP> at(t);
    const unsigned G = t.first[Table<S::NP>::N];
    const int lane = threadIdx.x & 63;
    const unsigned wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    d2 v[S::ROUNDS], x[S::ROUNDS], m[S::ROUNDS];
#pragma unroll
    for (int r = 0; r < S::ROUNDS; ++r) {
        const unsigned q = wave + r * SMALL_WAVES;
        if (q < G) {
            at.find(q, PIECE);
            const int i = (int)(q - at.f) * PIECE + 2 * lane, n = (int)at.n;
            v[r] = load_piece(at.p[S::READ], i, n);
            if (OP >= OP_SGD) x[r] = load_piece(at.p[0], i, n);
            if (OP == OP_SGD_MOMENTUM) m[r] = load_piece(at.p[S::NP - 1], i, n);
        }
    }
    Acc acc;
#pragma unroll
    for (int r = 0; r < S::ROUNDS; ++r)
        if (wave + r * SMALL_WAVES < G) add<CPLX>(acc, v[r]);
    const Norms nr = finish(reduce_block<SMALL_WAVES>(part_of<CPLX>(acc)), bd);
    if (threadIdx.x == 0) put_norms(nr, bd, ws);
    if (OP == OP_NORMS) return;
    scale(v, nr.k, bd.max_norm);
#pragma unroll
    for (int r = 0; r < S::ROUNDS; ++r) {
        const unsigned q = wave + r * SMALL_WAVES;
        if (q >= G) return;
        at.find(q, PIECE);
        const int i = (int)(q - at.f) * PIECE + 2 * lane, n = (int)at.n;
        if (OP == OP_CLIP) {
            if (nr.k != 1.0 || at.p[S::NP - 1] != at.p[0]) store_piece(v[r], at.p[S::NP - 1], i, n);
        } else {
            step_pair<OP == OP_SGD_MOMENTUM>(x[r], v[r], m[r], s);
            if (OP == OP_SGD_MOMENTUM) store_piece(v[r], at.p[S::NP - 1], i, n);
            store_piece(x[r], at.p[0], i, n);
        }
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------------------------

int list_error(ctm_ctx* ctx, const char* name, const std::string& what) {
    ctx->set_error(std::string(name) + ": " + what);
    return CTM_ERR_BADARG;
}

int check_device(ctm_ctx* ctx, const char* name) {
    int dev = -1;
    CTM_HIP_CHECK(ctx, hipGetDevice(&dev));
    if (dev != ctx->device) return list_error(ctx, name, "the context belongs to device " + std::to_string(ctx->device) + ", device " + std::to_string(dev) + " is current");
    return CTM_OK;
}

// launch on the caller's stream, CTM_LAUNCH's checks
#define GRADS_LAUNCH(ctx, stream, kernel, grid, block, ...)                                                       \
    do {                                                                                                          \
        if (g_ctm_sync_launch) ctm_note_launch(#kernel);                                                          \
        hipLaunchKernelGGL(kernel, dim3(grid), dim3(block), 0, stream, __VA_ARGS__);                              \
        hipError_t _le = hipGetLastError();                                                                       \
        if (_le == hipSuccess && g_ctm_sync_launch) _le = hipStreamSynchronize(stream);                           \
        if (_le != hipSuccess) {                                                                                  \
            (ctx)->set_error(std::string("launch of " #kernel ": ") + hipGetErrorString(_le));                    \
            return CTM_ERR_HIP;                                                                                   \
        }                                                                                                         \
    } while (0)

template <int OP> bool small(ctm_ctx* ctx, hipStream_t s, const Lists<Shape<OP>::NP>& L, const Size& z, Bound bd, const Step& st, double* ws, int* status) {
    Table<Shape<OP>::NP> t;
    if (z.tensors > t.N || z.pieces > Shape<OP>::ROUNDS * SMALL_WAVES) return false;
    if (fill(L, 0, t, PIECE) < L.nt) return false;       // (tensors too far from each other)
    *status = [&]() -> int {
        if (ctx->cplx) GRADS_LAUNCH(ctx, s, (small_kernel<OP, true>), 1, SMALL_THREADS, t, bd, st, ws);
        else GRADS_LAUNCH(ctx, s, (small_kernel<OP, false>), 1, SMALL_THREADS, t, bd, st, ws);
        return CTM_OK;
    }();
    return true;
}

// Lists that do not fit the 256 MB last-level cache are read by the norm pass without a claim on it (545 MB: 82 us against 87); stores of lists longer
// than the 32 MB of L2 cache bypass it (545 MB scaled in 185 us against 188 ... 229).
constexpr long long LLC_BYTES = 256LL << 20, L2_BYTES = 32LL << 20;

constexpr unsigned LONG = 8192;        // (4752 chunks clipped: 42.3 us joined by the workgroups, 43.7 with the kernel; 66560: 542 and 533)

// The norm pass, and where a second pass finds the factor (`last`: there is none, the norms are to be in ws)
int norm_pass(ctm_ctx* ctx, hipStream_t s, const Lists<1>& L, const Size& z, Bound bd, bool last, double* ws, Source* src) {
    Part* part = (Part*)(ws + WS_HEAD);
    int np = 0;
    for (int i = 0; i < L.nt;) {
        Table<1> t;
        i = fill(L, i, t);
        const unsigned g = t.first[t.N];
        if (!g) break;
        unsigned grid = PARTIALS_LEAST + (unsigned)((unsigned long long)PARTIALS * g / z.chunks);
        grid = grid > PARTIALS ? PARTIALS : grid;
        grid = grid > g ? g : grid;
        if (z.bytes > LLC_BYTES) {
            if (ctx->cplx) GRADS_LAUNCH(ctx, s, (norm_partials_kernel<true, true>), grid, THREADS, t, part + np);
            else GRADS_LAUNCH(ctx, s, (norm_partials_kernel<false, true>), grid, THREADS, t, part + np);
        } else {
            if (ctx->cplx) GRADS_LAUNCH(ctx, s, (norm_partials_kernel<true, false>), grid, THREADS, t, part + np);
            else GRADS_LAUNCH(ctx, s, (norm_partials_kernel<false, false>), grid, THREADS, t, part + np);
        }
        np += (int)grid;
    }
    const bool finish = last || z.chunks > LONG;
    if (finish) GRADS_LAUNCH(ctx, s, norm_finish_kernel, 1, 1024, (const Part*)part, np, bd, ws);
    *src = Source{part, finish ? 0 : np, bd, ws, !finish};
    return CTM_OK;
}

// Second pass over a list: launch(table, workgroups, source) for every table of it.  One workgroup per chunk: the table's lookup costs
// less than the tail of a grid that walks (1.1 GB clipped: 535 us against 553 with 8192 workgroups, 569 with 2048).
constexpr unsigned MOST = 1u << 23;          // (a grid holds at most 2^32 threads)
template <int NP, class F> int second_pass(const Lists<NP>& L, Source src, F&& launch) {
    for (int i = 0; i < L.nt;) {
        Table<NP> t;
        i = fill(L, i, t);
        const unsigned g = t.first[t.N];
        if (!g) break;
        CTM_TRY(launch(t, g < MOST ? g : MOST, src));
        src.write = false;                   // the norms are written once
    }
    return CTM_OK;
}

template <bool MOMENTUM> int sgd(ctm_ctx* ctx, hipStream_t s, const Lists<MOMENTUM ? 3 : 2>& L, const Size& z, const Step& st, const Source& src) {
    return second_pass(L, src, [&](const Table<MOMENTUM ? 3 : 2>& t, unsigned grid, const Source& f) -> int {
        if (z.bytes > L2_BYTES) GRADS_LAUNCH(ctx, s, (sgd_kernel<MOMENTUM, true>), grid, THREADS, t, st, f);
        else GRADS_LAUNCH(ctx, s, (sgd_kernel<MOMENTUM, false>), grid, THREADS, t, st, f);
        return CTM_OK;
    });
}

}  // namespace

extern "C" {

int ctm_grad_norms(ctm_ctx* ctx, void* hip_stream, int nt, const double* const* x, const long long* n, double* ws, long long ws_doubles) {
    return ctm_entry(ctx, "ctm_grad_norms", [&]() -> int {
    CTM_TRY(check_device(ctx, "grad_norms"));
    const bool written[1] = {false};
    if (const std::string e = check_lists(Lists<1>{nt, {x}, n, ctx->cplx ? 2 : 1}, written, 0); !e.empty()) return list_error(ctx, "grad_norms", e);
    if (!ws || ws_doubles < CTM_GRAD_WS_DOUBLES((long long)nt)) return list_error(ctx, "grad_norms", "workspace too small (CTM_GRAD_WS_DOUBLES)");
    hipStream_t s = (hipStream_t)hip_stream;
    const Lists<1> L{nt, {x}, n, ctx->cplx ? 2 : 1};
    const Size z = size_of(n, nt, L.unit);
    const Bound none{-1.0, 0};
    int status;
    if (small<OP_NORMS>(ctx, s, L, z, none, Step{}, ws, &status)) return status;
    Source src;
    return norm_pass(ctx, s, L, z, none, true, ws, &src);
    });
}

int ctm_grad_clip(ctm_ctx* ctx, void* hip_stream, int nt, const double* const* x, double* const* y, const long long* n, int norm_type,
                  double max_norm, double* ws, long long ws_doubles) {
    return ctm_entry(ctx, "ctm_grad_clip", [&]() -> int {
    CTM_TRY(check_device(ctx, "grad_clip"));
    const bool written[2] = {false, true};
    Lists<2> L{nt, {x, (const double* const*)y}, n, ctx->cplx ? 2 : 1};
    if (const std::string e = check_lists(L, written, 1); !e.empty()) return list_error(ctx, "grad_clip", e);
    if (!(max_norm >= 0.0)) return list_error(ctx, "grad_clip", "max_norm must be >= 0");
    if (norm_type != CTM_NORM_2 && norm_type != CTM_NORM_INF) return list_error(ctx, "grad_clip", "norm_type must be CTM_NORM_2 or CTM_NORM_INF");
    if (!ws || ws_doubles < CTM_GRAD_WS_DOUBLES((long long)nt)) return list_error(ctx, "grad_clip", "workspace too small (CTM_GRAD_WS_DOUBLES)");
    hipStream_t s = (hipStream_t)hip_stream;
    const Bound bd{max_norm, norm_type == CTM_NORM_INF};
    const Size z = size_of(n, nt, L.unit);
    int status;
    Source src;
    if (small<OP_CLIP>(ctx, s, L, z, bd, Step{}, ws, &status)) return status;
    CTM_TRY(norm_pass(ctx, s, Lists<1>{nt, {x}, n, L.unit}, z, bd, false, ws, &src));
    return second_pass(L, src, [&](const Table<2>& t, unsigned grid, const Source& f) -> int {
        if (z.bytes > L2_BYTES) GRADS_LAUNCH(ctx, s, clip_kernel<true>, grid, THREADS, t, f);
        else GRADS_LAUNCH(ctx, s, clip_kernel<false>, grid, THREADS, t, f);
        return CTM_OK;
    });
    });
}

int ctm_sgd_step(ctm_ctx* ctx, void* hip_stream, int nt, double* const* p, const double* const* g, double* const* m, const long long* n,
                 double lr, double momentum, double dampening, int first, int norm_type, double max_norm, double* ws, long long ws_doubles) {
    return ctm_entry(ctx, "ctm_sgd_step", [&]() -> int {
    CTM_TRY(check_device(ctx, "sgd_step"));
    Lists<3> L3{nt, {(const double* const*)p, g, (const double* const*)m}, n, ctx->cplx ? 2 : 1};
    Lists<2> L2{nt, {(const double* const*)p, g}, n, ctx->cplx ? 2 : 1};
    const bool w3[3] = {true, false, true}, w2[2] = {true, false};
    if (const std::string e = m ? check_lists(L3, w3, 0) : check_lists(L2, w2, 0); !e.empty()) return list_error(ctx, "sgd_step", e);
    if (nt > 0 && !m && momentum != 0.0) return list_error(ctx, "sgd_step", "momentum needs the momentum buffers");
    hipStream_t s = (hipStream_t)hip_stream;
    const bool bounded = max_norm >= 0.0;
    if (max_norm != max_norm) return list_error(ctx, "sgd_step", "max_norm is NaN");
    if (bounded) {
        if (norm_type != CTM_NORM_2 && norm_type != CTM_NORM_INF) return list_error(ctx, "sgd_step", "norm_type must be CTM_NORM_2 or CTM_NORM_INF");
        if (!ws || ws_doubles < CTM_GRAD_WS_DOUBLES((long long)nt)) return list_error(ctx, "sgd_step", "workspace too small (CTM_GRAD_WS_DOUBLES)");
    }
    const Step st{lr, momentum, 1.0 - dampening, first};
    const Size z = size_of(n, nt, L2.unit);
    const Bound bd{bounded ? max_norm : -1.0, norm_type == CTM_NORM_INF};
    Source src{nullptr, 0, bd, ws, false};
    if (bounded) {
        int status;
        if (m ? small<OP_SGD_MOMENTUM>(ctx, s, L3, z, bd, st, ws, &status) : small<OP_SGD>(ctx, s, L2, z, bd, st, ws, &status)) return status;
        CTM_TRY(norm_pass(ctx, s, Lists<1>{nt, {g}, n, L2.unit}, z, bd, false, ws, &src));
    }
    return m ? sgd<true>(ctx, s, L3, z, st, src) : sgd<false>(ctx, s, L2, z, st, src);
    });
}

}  // extern "C"
