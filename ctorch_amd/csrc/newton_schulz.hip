// Orthogonalised updates: Newton-Schulz products on the f16 matrix cores, and the optimiser step around
// them.
//   X = U / (|U|_F + eps), transposed if that makes it wide (m rows, n columns, m <= n); `steps` times
//     A = X X^T,  B = b A + c A A,  X = a X + B X
// drives the singular values of U towards one; three products a step, two of them symmetric.
//
// Bound by the matrix cores.  fp32 MFMA runs at 1 / 16 of the f16 rate, so every matrix is kept as a pair
// of f16 numbers, x = (hi + lo) / scale: hi is x rounded to 11 bits, lo the rest rounded to 11 bits, 22 bits
// together in the 32 that a float takes.  A product is three MFMAs with fp32 accumulation,
//   hi hi' + hi lo' + lo hi',
// what is left out (lo lo') is below 2^-22 of the terms, as is the rounding of the pair.  Against 64 bits the
// iteration ends where the one in fp32 products does (2.4e-6 of the largest entry for both at 1024 x 1024):
// the polynomial's slope at zero, a^steps, magnifies any rounding of the first steps alike.
//
// Layout of a matrix of pairs: row-major, rows padded to 64 columns (zeros), each run of 8 columns stored as
// [8 hi][8 lo], 32 bytes.  A k step of 32 is 128 bytes of a row, one cache line, and goes to LDS by the
// direct-to-LDS load; 16-byte units are permuted by the row's low bits so that the fragment reads (one
// ds_read_b128 per 32 x 16 operand half) meet no bank twice.  Both operands of every product are read
// along their rows (A and B are symmetric; X is kept with its transpose Y), so one kernel serves all three.
#include <cmath>

#include "common.h"

namespace ctamd {
namespace {

typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kXcds = 8;
// X and Y are stored times 2^13 (entries up to 8), A and B times 2^11 (up to 32)
constexpr float kScaleX = 8192.0f, kScaleA = 2048.0f;

constexpr int kMaxJobs = 16;
constexpr int kNormParts = 256;

// One matrix - or `count` matrices of one shape, `stride` elements apart - of a call.
struct Job {
    const float* grad;
    const float* momentum;       // null: the update is the gradient itself
    const float* param;          // null: the result is the orthogonalised matrix itself
    float* new_momentum;
    float* out;                  // new parameter or orthogonalised matrix
    char* work;                  // workspace of the first matrix
    size_t stride, work_stride;  // elements, bytes
    int64_t rows, cols;
    int m, n, mp, np;            // min and max of rows, cols; padded to 64
    unsigned count;
    int tall;                    // rows > cols: X is the transposed update
    float step;                  // learning rate times the matrix's scale
    unsigned norm_parts;
    size_t part_size;            // elements per part of the norm
};
struct Table {
    int jobs;
    unsigned first[kMaxJobs + 1];     // first block of each job in this launch
    Job job[kMaxJobs];
    float mu, decay, eps;
    int nesterov;
};

// workspace of one matrix: the norm's partial sums, X and Y twice, A, B
__host__ __device__ inline size_t pairs_xy(const Job& j) { return size_t(j.mp) * j.np * 4; }
__host__ __device__ inline size_t pairs_a(const Job& j) { return size_t(j.mp) * j.mp * 4; }
constexpr size_t kNormBytes = kNormParts * sizeof(double);
__device__ inline char* buf_x(const Job& j, char* w, int which) { return w + kNormBytes + size_t(which) * 2 * pairs_xy(j); }
__device__ inline char* buf_y(const Job& j, char* w, int which) { return w + kNormBytes + (size_t(which) * 2 + 1) * pairs_xy(j); }
__device__ inline char* buf_a(const Job& j, char* w) { return w + kNormBytes + 4 * pairs_xy(j); }
__device__ inline char* buf_b(const Job& j, char* w) { return w + kNormBytes + 4 * pairs_xy(j) + pairs_a(j); }

__device__ __forceinline__ int job_of(const Table& t, unsigned block) {
    int j = 0;
    while (j + 1 < t.jobs && block >= t.first[j + 1]) ++j;
    return j;
}

// block-wide sum in a fixed order (kThreads threads); the result is valid in every thread
__device__ __forceinline__ double block_sum(double v, double* s_part) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if ((threadIdx.x & 63) == 0) s_part[threadIdx.x >> 6] = v;
    __syncthreads();
    return (s_part[0] + s_part[1]) + (s_part[2] + s_part[3]);
}

// The new momentum, and the sums of squares of the update u: parts in double, so that no gradient is too
// large or too small for its norm.
__global__ __launch_bounds__(kThreads) void momentum_norm(Table t) {
    __shared__ double s_part[kThreads / 64];
    const Job& j = t.job[job_of(t, blockIdx.x)];
    const unsigned local = blockIdx.x - t.first[job_of(t, blockIdx.x)], item = local / j.norm_parts, part = local % j.norm_parts;
    const size_t elements = size_t(j.rows) * j.cols, first = size_t(part) * j.part_size;
    size_t last = first + j.part_size;
    if (last > elements) last = elements;
    const float* g = j.grad + item * j.stride;
    double sum = 0.0;
    if (j.momentum) {
        const float* mo = j.momentum + item * j.stride;
        float* mn = j.new_momentum + item * j.stride;
        for (size_t i = first + threadIdx.x; i < last; i += kThreads) {
            const float gi = g[i], m = t.mu * mo[i] + gi;
            mn[i] = m;
            const double u = t.nesterov ? gi + t.mu * m : m;
            sum += u * u;
        }
    } else {
        for (size_t i = first + threadIdx.x; i < last; i += kThreads) {
            const double u = g[i];
            sum += u * u;
        }
    }
    sum = block_sum(sum, s_part);
    if (threadIdx.x == 0) reinterpret_cast<double*>(j.work + item * j.work_stride)[part] = sum;
}

// 1 / (|U|_F + eps) from the parts; every thread gets it.  Kept in double: its product with an element of U
// is rounded once, and a norm of 1e38 has an inverse.
__device__ __forceinline__ double inverse_norm(const Table& t, const Job& j, const char* work, double* s_part) {
    const double v = threadIdx.x < j.norm_parts ? reinterpret_cast<const double*>(work)[threadIdx.x] : 0.0;
    return 1.0 / (sqrt(block_sum(v, s_part)) + double(t.eps));
}
static_assert(kNormParts <= kThreads, "a thread per part");

__device__ __forceinline__ float update_at(const Table& t, const Job& j, size_t i) {
    if (!j.momentum) return j.grad[i];
    const float m = j.new_momentum[i];
    return t.nesterov ? j.grad[i] + t.mu * m : m;
}

__device__ __forceinline__ void split8(const float (&v)[8], float scale, h8* hi, h8* lo) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float s = v[e] * scale;
        const _Float16 h = _Float16(s);
        (*hi)[e] = h;
        (*lo)[e] = _Float16(s - float(h));
    }
}

// Divides the update by its norm and writes it as pairs, straight and transposed; a block per 64 x 64 tile.
__global__ __launch_bounds__(kThreads) void load_pairs(Table t) {
    __shared__ double s_part[kThreads / 64];
    __shared__ float s_tile[64][65];
    const int which = job_of(t, blockIdx.x);
    const Job& j = t.job[which];
    const unsigned local = blockIdx.x - t.first[which];
    const unsigned rp = unsigned(j.tall ? j.np : j.mp), cp = unsigned(j.tall ? j.mp : j.np);     // padded rows, columns of the update
    const unsigned tiles = (rp / 64) * (cp / 64), item = local / tiles, tile = local % tiles;
    const unsigned r0 = (tile / (cp / 64)) * 64, c0 = (tile % (cp / 64)) * 64;
    char* work = j.work + item * j.work_stride;
    const double inv = inverse_norm(t, j, work, s_part);
    char* straight = j.tall ? buf_y(j, work, 0) : buf_x(j, work, 0);
    char* turned = j.tall ? buf_x(j, work, 0) : buf_y(j, work, 0);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const unsigned r = (threadIdx.x >> 3) + 32 * q, c = (threadIdx.x & 7) * 8;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool in = int64_t(r0 + r) < j.rows && int64_t(c0 + c + e) < j.cols;
            v[e] = in ? float(update_at(t, j, item * j.stride + size_t(r0 + r) * j.cols + c0 + c + e) * inv) : 0.0f;
            s_tile[r][c + e] = v[e];
        }
        h8 hi, lo;
        split8(v, kScaleX, &hi, &lo);
        h8* dst = reinterpret_cast<h8*>(straight + (size_t(r0 + r) * cp + c0 + c) * 4);
        dst[0] = hi;
        dst[1] = lo;
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const unsigned c = (threadIdx.x >> 3) + 32 * q, r = (threadIdx.x & 7) * 8;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = s_tile[r + e][c];
        h8 hi, lo;
        split8(v, kScaleX, &hi, &lo);
        h8* dst = reinterpret_cast<h8*>(turned + (size_t(c0 + c) * rp + r0 + r) * 4);
        dst[0] = hi;
        dst[1] = lo;
    }
}

__device__ __forceinline__ float result_at(const Table& t, const Job& j, size_t i, float o) {
    return j.param ? j.param[i] * t.decay - j.step * o : o;
}

// steps == 0: the normalised update is the result
__global__ __launch_bounds__(kThreads) void scaled_update(Table t) {
    __shared__ double s_part[kThreads / 64];
    const int which = job_of(t, blockIdx.x);
    const Job& j = t.job[which];
    const unsigned local = blockIdx.x - t.first[which], item = local / j.norm_parts, part = local % j.norm_parts;
    const double inv = inverse_norm(t, j, j.work + item * j.work_stride, s_part);
    const size_t elements = size_t(j.rows) * j.cols, first = size_t(part) * j.part_size;
    size_t last = first + j.part_size;
    if (last > elements) last = elements;
    for (size_t i = first + threadIdx.x; i < last; i += kThreads) {
        const size_t at = item * j.stride + i;
        j.out[at] = result_at(t, j, at, float(update_at(t, j, at) * inv));
    }
}

// ------------------------------------------------------------------------------- the product
// GRAM: A = X X^T.  POLY: B = b A + c A A.  STEP: X' = a X + B X, and Y' its transpose.  LAST: the same,
// written as the call's result.
enum Kind { GRAM, POLY, STEP, LAST };

template <int BT_, int WM_, int WN_>
struct TileCfg {
    static constexpr int BT = BT_, WM = WM_, WN = WN_;         // square block tile, wave tile
    static constexpr int TM = WM / 32, TN = WN / 32;
    static constexpr int WAVES = (BT / WM) * (BT / WN), THREADS = WAVES * 64;
    static constexpr int BUF = 2 * BT * 128;                   // bytes of one k step of both operands
    static constexpr int LOADS = 2 * BT / (WAVES * 8);         // direct-to-LDS loads per wave and k step
    static_assert(BT % (WAVES * 8) == 0, "a load does not straddle the operands");
    static_assert(WAVES * 4096 <= BUF, "the epilogue turns a 32 x 32 tile per wave in one buffer");
};

__device__ __forceinline__ void lds_load(const char* g, char* l) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g, (__attribute__((address_space(3))) void*)l, 16, 0, 0);
}

template <class C, Kind KIND>
__global__ __launch_bounds__(C::THREADS) void pair_product(Table t, int from, float ca, float cb, float cc) {
    __shared__ __attribute__((aligned(128))) char s_buf0[C::BUF];
    __shared__ __attribute__((aligned(128))) char s_buf1[C::BUF];
    const int which = job_of(t, blockIdx.x);
    const Job& j = t.job[which];
    const unsigned here = t.first[which + 1] - t.first[which];
    unsigned local = blockIdx.x - t.first[which];
    // blocks go to the XCDs in turn: give each XCD a run of neighbouring tiles, which share operand rows in its L2
    const unsigned q8 = here / kXcds, r8 = here % kXcds, xcd = local % kXcds;
    local = xcd * q8 + (xcd < r8 ? xcd : r8) + local / kXcds;
    const unsigned tm = (unsigned(j.mp) + C::BT - 1) / C::BT, tn = (unsigned(j.np) + C::BT - 1) / C::BT;
    constexpr bool SYM = KIND == GRAM || KIND == POLY;
    const unsigned tiles = SYM ? tm * (tm + 1) / 2 : tm * tn;
    const unsigned item = local / tiles, tile = local % tiles;
    unsigned ti, tj;
    if (SYM) {                                       // tile = ti (ti + 1) / 2 + tj, tj <= ti
        ti = unsigned((sqrtf(8.0f * float(tile) + 1.0f) - 1.0f) * 0.5f);
        while (ti * (ti + 1) / 2 > tile) --ti;
        while ((ti + 1) * (ti + 2) / 2 <= tile) ++ti;
        tj = tile - ti * (ti + 1) / 2;
    } else {
        tj = tile / tm;
        ti = tile % tm;
    }
    char* work = j.work + item * j.work_stride;
    const char* p = KIND == GRAM ? buf_x(j, work, from) : KIND == POLY ? buf_a(j, work) : buf_b(j, work);
    const char* q = KIND == GRAM ? buf_x(j, work, from) : KIND == POLY ? buf_a(j, work) : buf_y(j, work, from);
    const unsigned k = unsigned(KIND == GRAM ? j.np : j.mp);
    const unsigned rows_p = unsigned(j.mp), rows_q = unsigned(SYM ? j.mp : j.np);
    const unsigned i0 = ti * C::BT, j0 = tj * C::BT;

    const unsigned wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    // this lane's byte offset of every load, from the operand's first row of the tile; rows beyond the matrix
    // read its last one (their results are not stored)
    unsigned off[C::LOADS];
#pragma unroll
    for (int l = 0; l < C::LOADS; ++l) {
        unsigned r = unsigned(l) * C::WAVES * 8 + wave * 8 + (lane >> 3);
        const bool second = l >= C::LOADS / 2;
        if (second) r -= C::BT;
        const unsigned most = (second ? rows_q - j0 : rows_p - i0) - 1;
        if (r > most) r = most;
        off[l] = r * k * 4 + ((lane & 7) ^ (lane >> 3)) * 16;
    }
    const char* pb = p + size_t(i0) * k * 4;
    const char* qb = q + size_t(j0) * k * 4;
    auto load = [&](char* buf, unsigned step) {
#pragma unroll
        for (int l = 0; l < C::LOADS; ++l)
            lds_load((l < C::LOADS / 2 ? pb : qb) + size_t(step) * 128 + off[l], buf + (l * C::WAVES + wave) * 1024);
        __builtin_amdgcn_sched_barrier(0);
    };

    const unsigned wm = (wave / (C::BT / C::WN)) * C::WM, wn = (wave % (C::BT / C::WN)) * C::WN;
    v16f acc[C::TM][C::TN];
#pragma unroll
    for (int a = 0; a < C::TM; ++a)
#pragma unroll
        for (int b = 0; b < C::TN; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[a][b][e] = 0.0f;
    auto multiply = [&](const char* buf) {
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            h8 fp[C::TM][2], fq[C::TN][2];
            const unsigned unit = (kk * 2 + (lane >> 5)) * 2, r = lane & 31;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const unsigned at = r * 128 + (((unit + h) ^ (r & 7)) * 16);
#pragma unroll
                for (int a = 0; a < C::TM; ++a) fp[a][h] = *reinterpret_cast<const h8*>(buf + (wm + a * 32) * 128 + at);
#pragma unroll
                for (int b = 0; b < C::TN; ++b) fq[b][h] = *reinterpret_cast<const h8*>(buf + (C::BT + wn + b * 32) * 128 + at);
            }
#pragma unroll
            for (int a = 0; a < C::TM; ++a)
#pragma unroll
                for (int b = 0; b < C::TN; ++b) {
                    acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[a][0], fq[b][0], acc[a][b], 0, 0, 0);
                    acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[a][0], fq[b][1], acc[a][b], 0, 0, 0);
                    acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[a][1], fq[b][0], acc[a][b], 0, 0, 0);
                }
        }
    };
    const unsigned steps = k / 32;                   // even: k is a multiple of 64
    load(s_buf0, 0);
    __syncthreads();
    for (unsigned s = 0; s < steps; s += 2) {
        load(s_buf1, s + 1);
        multiply(s_buf0);
        __syncthreads();
        if (s + 2 < steps) load(s_buf0, s + 2);
        multiply(s_buf1);
        __syncthreads();
    }

    // accumulator register e of a lane: row 8 (e / 4) + 4 (lane / 32) + e % 4, column lane % 32 of its 32 x 32 tile
    const bool mirror = !SYM || ti != tj;            // a tile on the diagonal is its own mirror image
    const unsigned ld_direct = SYM ? rows_p : rows_q, ld_turned = rows_p;
    char* direct = KIND == GRAM ? buf_a(j, work) : KIND == POLY ? buf_b(j, work) : buf_x(j, work, from ^ 1);
    char* turned = KIND == GRAM ? buf_a(j, work) : KIND == POLY ? buf_b(j, work) : buf_y(j, work, from ^ 1);
    const char* addend = KIND == POLY ? buf_a(j, work) : buf_y(j, work, from);
    uint32_t* s_turn = reinterpret_cast<uint32_t*>(s_buf0) + wave * 1024;
    const unsigned half = lane >> 5, col = lane & 31;
#pragma unroll
    for (int a = 0; a < C::TM; ++a)
#pragma unroll
        for (int b = 0; b < C::TN; ++b) {
            const unsigned gi = i0 + wm + a * 32, gj = j0 + wn + b * 32;
            if (gi >= rows_p || gj >= rows_q) continue;                        // wave-uniform; rows are multiples of 64
#pragma unroll
            for (int quad = 0; quad < 4; ++quad) {
                const size_t at = (size_t(gj + col) * ld_turned + gi) * 4 + quad * 32 + half * 8;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = acc[a][b][quad * 4 + e];
                if (KIND == GRAM) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] *= kScaleA / (kScaleX * kScaleX);
                } else {
                    const h4 oh = *reinterpret_cast<const h4*>(addend + at), ol = *reinterpret_cast<const h4*>(addend + at + 16);
                    const float f = KIND == POLY ? cc / kScaleA : KIND == STEP ? 1.0f / kScaleA : 1.0f / (kScaleA * kScaleX);
                    const float old = KIND == POLY ? cb : KIND == STEP ? ca : ca / kScaleX;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = v[e] * f + old * (float(oh[e]) + float(ol[e]));
                }
                if (KIND == LAST) {
                    const unsigned x0 = gi + quad * 8 + half * 4, y = gj + col;
                    if (y < unsigned(j.n)) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (x0 + e < unsigned(j.m)) {
                                const size_t o = item * j.stride + (j.tall ? size_t(y) * j.cols + x0 + e : size_t(x0 + e) * j.cols + y);
                                j.out[o] = result_at(t, j, o, v[e]);
                            }
                    }
                    continue;
                }
                h4 hi, lo;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    hi[e] = _Float16(v[e]);
                    lo[e] = _Float16(v[e] - float(hi[e]));
                    const unsigned row = quad * 8 + half * 4 + e;
                    const uint32_t word = uint32_t(__builtin_bit_cast(uint16_t, _Float16(hi[e]))) |
                                          (uint32_t(__builtin_bit_cast(uint16_t, _Float16(lo[e]))) << 16);
                    s_turn[row * 32 + ((((col >> 2) ^ row) & 7) << 2) + (col & 3)] = word;
                }
                if (mirror) {
                    *reinterpret_cast<h4*>(turned + at) = hi;
                    *reinterpret_cast<h4*>(turned + at + 16) = lo;
                }
            }
            if (KIND == LAST) continue;
            // a wave reads back only what it wrote itself
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const unsigned row = (lane >> 2) + 16 * h, c8 = lane & 3;
                const u4 w0 = *reinterpret_cast<const u4*>(s_turn + row * 32 + (((2 * c8) ^ row) & 7) * 4);
                const u4 w1 = *reinterpret_cast<const u4*>(s_turn + row * 32 + (((2 * c8 + 1) ^ row) & 7) * 4);
                u4 hi, lo;
                hi[0] = (w0[0] & 0xffffu) | (w0[1] << 16);
                hi[1] = (w0[2] & 0xffffu) | (w0[3] << 16);
                hi[2] = (w1[0] & 0xffffu) | (w1[1] << 16);
                hi[3] = (w1[2] & 0xffffu) | (w1[3] << 16);
                lo[0] = (w0[0] >> 16) | (w0[1] & 0xffff0000u);
                lo[1] = (w0[2] >> 16) | (w0[3] & 0xffff0000u);
                lo[2] = (w1[0] >> 16) | (w1[1] & 0xffff0000u);
                lo[3] = (w1[2] >> 16) | (w1[3] & 0xffff0000u);
                u4* dst = reinterpret_cast<u4*>(direct + (size_t(gi + row) * ld_direct + gj + c8 * 8) * 4);
                dst[0] = hi;
                dst[1] = lo;
            }
            __builtin_amdgcn_wave_barrier();
        }
}

// ------------------------------------------------------------------------------- host side
constexpr int64_t kMostExtent = int64_t(1) << 20, kMostSide = int64_t(1) << 15;
constexpr int kMostSteps = 64;
constexpr float kCoefficients[3] = {3.4445f, -4.7750f, 2.0315f};

int check_matrix(const char* who, int64_t rows, int64_t cols) {
    if (rows < 0 || cols < 0) return fail(CTAMD_EINVAL, "%s: negative extent", who);
    if (rows > kMostExtent || cols > kMostExtent || (rows > kMostSide && cols > kMostSide))
        return fail(CTAMD_ERANGE, "%s: %lld x %lld: at most 2^20, and 2^15 on the shorter side", who, (long long)rows, (long long)cols);
    return CTAMD_OK;
}
int check_iteration(const char* who, int steps, const float* c, float eps) {
    if (steps < 0 || steps > kMostSteps) return fail(CTAMD_EINVAL, "%s: %d steps, 0 to %d", who, steps, kMostSteps);
    for (int i = 0; i < 3; ++i)
        if (!(std::fabs(c[i]) <= 32.0f)) return fail(CTAMD_EINVAL, "%s: a coefficient beyond 32", who);
    if (!(eps >= 0.0f)) return fail(CTAMD_EINVAL, "%s: eps must not be negative", who);
    return CTAMD_OK;
}

void shape_job(Job* j, int64_t rows, int64_t cols, unsigned count) {
    j->rows = rows;
    j->cols = cols;
    j->tall = rows > cols;
    j->m = int(rows < cols ? rows : cols);
    j->n = int(rows < cols ? cols : rows);
    j->mp = (j->m + 63) / 64 * 64;
    j->np = (j->n + 63) / 64 * 64;
    j->count = count;
    j->stride = size_t(rows) * size_t(cols);
    size_t size = (j->stride + kNormParts - 1) / kNormParts;
    if (size < 4096) size = 4096;
    j->part_size = size;
    j->norm_parts = unsigned((j->stride + size - 1) / size);
    j->work_stride = kNormBytes + 4 * pairs_xy(*j) + 2 * pairs_a(*j);
}

typedef TileCfg<64, 32, 32> Tile64;
typedef TileCfg<128, 64, 64> Tile128;
typedef TileCfg<256, 128, 64> Tile256;

double flops_of(const Job& j, int steps) {
    const double m = j.m, n = j.n;
    return j.count * steps * (m * (m + 1) * n + m * (m + 1) * m + 2 * m * m * n);
}

// Lays the jobs' blocks out for a launch and returns their number; per(job) blocks for each matrix
template <class F>
unsigned lay_out(Table* t, F per) {
    t->first[0] = 0;
    for (int j = 0; j < t->jobs; ++j) t->first[j + 1] = t->first[j] + t->job[j].count * per(t->job[j]);
    return t->first[t->jobs];
}

template <class C>
int iterate(const char* who, Table* t, int steps, const float* c, hipStream_t s) {
    auto sym = [](const Job& j) {
        const unsigned tm = (unsigned(j.mp) + C::BT - 1) / C::BT;
        return tm * (tm + 1) / 2;
    };
    auto full = [](const Job& j) { return ((unsigned(j.mp) + C::BT - 1) / C::BT) * ((unsigned(j.np) + C::BT - 1) / C::BT); };
    for (int k = 0; k < steps; ++k) {
        const int from = k & 1;
        unsigned blocks = lay_out(t, sym);
        hipLaunchKernelGGL((pair_product<C, GRAM>), dim3(blocks), dim3(C::THREADS), 0, s, *t, from, c[0], c[1], c[2]);
        hipLaunchKernelGGL((pair_product<C, POLY>), dim3(blocks), dim3(C::THREADS), 0, s, *t, from, c[0], c[1], c[2]);
        blocks = lay_out(t, full);
        if (k + 1 < steps) hipLaunchKernelGGL((pair_product<C, STEP>), dim3(blocks), dim3(C::THREADS), 0, s, *t, from, c[0], c[1], c[2]);
        else hipLaunchKernelGGL((pair_product<C, LAST>), dim3(blocks), dim3(C::THREADS), 0, s, *t, from, c[0], c[1], c[2]);
        const int rc = launched(who);
        if (rc) return rc;
    }
    return CTAMD_OK;
}

int run_table(const char* who, Table* t, int steps, const float* c, hipStream_t s) {
    if (!t->jobs) return CTAMD_OK;
    double bytes = 0, flops = 0;
    for (int j = 0; j < t->jobs; ++j) {
        bytes += (t->job[j].param ? 20.0 : 8.0) * double(t->job[j].stride) * t->job[j].count;
        flops += flops_of(t->job[j], steps);
    }
    unsigned blocks = lay_out(t, [](const Job& j) { return j.norm_parts; });
    hipLaunchKernelGGL(momentum_norm, dim3(blocks), dim3(kThreads), 0, s, *t);
    int rc = launched(who);
    if (rc) return rc;
    if (steps == 0) {
        hipLaunchKernelGGL(scaled_update, dim3(blocks), dim3(kThreads), 0, s, *t);
        rc = launched(who);
    } else {
        blocks = lay_out(t, [](const Job& j) { return unsigned(j.mp / 64) * unsigned(j.np / 64); });
        hipLaunchKernelGGL(load_pairs, dim3(blocks), dim3(kThreads), 0, s, *t);
        rc = launched(who);
        if (rc) return rc;
        const size_t cus = size_t(compute_units() > 0 ? compute_units() : 256);
        size_t at256 = 0, at128 = 0;
        for (int j = 0; j < t->jobs; ++j) {
            const Job& b = t->job[j];
            at256 += size_t(b.count) * ((b.mp + 255) / 256) * ((b.np + 255) / 256);
            at128 += size_t(b.count) * ((b.mp + 127) / 128) * ((b.np + 127) / 128);
        }
        rc = at256 >= cus * 3 / 4 ? iterate<Tile256>(who, t, steps, c, s)
             : at128 >= cus * 3 / 4 ? iterate<Tile128>(who, t, steps, c, s) : iterate<Tile64>(who, t, steps, c, s);
    }
    if (!rc) account(bytes, flops);
    return rc;
}

// What one table takes: block counts that fit a launch, and a workspace of 2 GiB (a larger matrix has a
// table of its own); longer calls take several tables, one after the other in the same workspace.
constexpr size_t kMostTiles = size_t(1) << 22, kMostWork = size_t(2) << 30;
size_t tiles_of(const Job& j) { return size_t(j.mp / 64) * size_t(j.np / 64); }
int64_t batch_at_once(const Job& j) {
    const size_t a = kMostTiles / tiles_of(j), b = kMostWork / j.work_stride, c = a < b ? a : b;
    return c > 0 ? int64_t(c) : 1;
}

}  // namespace
}  // namespace ctamd

using namespace ctamd;

extern "C" {

int ctamd_newton_schulz_workspace(int64_t rows, int64_t cols, int64_t batch, size_t* bytes_host) {
    if (!bytes_host) return fail(CTAMD_EINVAL, "%s: null output", __func__);
    *bytes_host = 0;
    int rc = check_matrix(__func__, rows, cols);
    if (rc) return rc;
    if (batch < 0) return fail(CTAMD_EINVAL, "%s: negative batch", __func__);
    if (rows == 0 || cols == 0 || batch == 0) return CTAMD_OK;
    Job j{};
    shape_job(&j, rows, cols, 1);
    const int64_t at_once = batch_at_once(j);
    *bytes_host = j.work_stride * size_t(batch < at_once ? batch : at_once);
    return CTAMD_OK;
}

int ctamd_newton_schulz_f32(const float* g, float* out, int64_t rows, int64_t cols, int64_t batch, int steps, const float* coefficients_host,
                            float eps, void* workspace, size_t workspace_bytes, void* stream) {
    const float* c = coefficients_host ? coefficients_host : kCoefficients;
    int rc = check_matrix(__func__, rows, cols);
    if (!rc) rc = check_iteration(__func__, steps, c, eps);
    if (rc) return rc;
    if (batch < 0) return fail(CTAMD_EINVAL, "%s: negative batch", __func__);
    if (rows == 0 || cols == 0 || batch == 0) return CTAMD_OK;
    if (!g || !out) return fail(CTAMD_EINVAL, "%s: null pointer", __func__);
    size_t need = 0;
    rc = ctamd_newton_schulz_workspace(rows, cols, batch, &need);
    if (rc) return rc;
    if (!workspace || workspace_bytes < need || !aligned16(workspace))
        return fail(CTAMD_EINVAL, "%s: a workspace of %zu bytes, 16-byte aligned, is needed", __func__, need);
    Table t{};
    t.eps = eps;
    Job& j = t.job[0];
    shape_job(&j, rows, cols, 1);
    const int64_t at_once = batch_at_once(j);
    for (int64_t done = 0; done < batch; done += at_once) {
        t.jobs = 1;
        j.count = unsigned(batch - done < at_once ? batch - done : at_once);
        j.grad = g + size_t(done) * j.stride;
        j.out = out + size_t(done) * j.stride;
        j.work = static_cast<char*>(workspace);
        rc = run_table(__func__, &t, steps, c, as_stream(stream));
        if (rc) return rc;
    }
    return CTAMD_OK;
}

// the matrices [*at, end) of a call that go into one table, laid out in the workspace; bytes they need there
static size_t next_table(const ctamd_muon_matrix* matrices, int count, int* at, Table* t, char* work, float lr) {
    size_t bytes = 0, tiles = 0;
    t->jobs = 0;
    for (; *at < count && t->jobs < kMaxJobs; ++*at) {
        const ctamd_muon_matrix& a = matrices[*at];
        if (a.rows == 0 || a.cols == 0) continue;
        Job& j = t->job[t->jobs];
        shape_job(&j, a.rows, a.cols, 1);
        if (t->jobs && (tiles + tiles_of(j) > kMostTiles || bytes + j.work_stride > kMostWork)) break;
        tiles += tiles_of(j);
        j.grad = a.grad;
        j.momentum = a.momentum;
        j.param = a.param;
        j.new_momentum = a.new_momentum;
        j.out = a.new_param;
        j.step = lr * a.scale;
        j.work = work ? work + bytes : nullptr;
        bytes += j.work_stride;
        ++t->jobs;
    }
    return bytes;
}

int ctamd_muon_workspace(const ctamd_muon_matrix* matrices, int count, size_t* bytes_host) {
    if (!bytes_host) return fail(CTAMD_EINVAL, "%s: null output", __func__);
    *bytes_host = 0;
    if (count < 0) return fail(CTAMD_EINVAL, "%s: negative count", __func__);
    if (count && !matrices) return fail(CTAMD_EINVAL, "%s: null table", __func__);
    for (int i = 0; i < count; ++i) {
        const int rc = check_matrix(__func__, matrices[i].rows, matrices[i].cols);
        if (rc) return rc;
    }
    Table t{};
    for (int at = 0; at < count;) {
        const size_t b = next_table(matrices, count, &at, &t, nullptr, 0.0f);
        if (b > *bytes_host) *bytes_host = b;
    }
    return CTAMD_OK;
}

int ctamd_muon_step_f32(const ctamd_muon_matrix* matrices, int count, const ctamd_muon_options* options, void* workspace, size_t workspace_bytes,
                        void* stream) {
    if (!options) return fail(CTAMD_EINVAL, "%s: null options", __func__);
    int rc = check_iteration(__func__, options->steps, options->coefficients, options->eps);
    if (rc) return rc;
    size_t need = 0;
    rc = ctamd_muon_workspace(matrices, count, &need);
    if (rc) return rc;
    for (int i = 0; i < count; ++i) {
        const ctamd_muon_matrix& a = matrices[i];
        if (a.rows && a.cols && (!a.param || !a.grad || !a.momentum || !a.new_param || !a.new_momentum))
            return fail(CTAMD_EINVAL, "%s: null tensor in matrix %d", __func__, i);
    }
    if (need && (!workspace || workspace_bytes < need || !aligned16(workspace)))
        return fail(CTAMD_EINVAL, "%s: a workspace of %zu bytes, 16-byte aligned, is needed", __func__, need);
    Table t{};
    t.mu = options->momentum;
    t.decay = 1.0f - options->learning_rate * options->weight_decay;
    t.eps = options->eps;
    t.nesterov = options->nesterov != 0;
    for (int at = 0; at < count;) {
        (void)next_table(matrices, count, &at, &t, static_cast<char*>(workspace), options->learning_rate);
        rc = run_table(__func__, &t, options->steps, options->coefficients, as_stream(stream));
        if (rc) return rc;
    }
    return CTAMD_OK;
}

}  // extern "C"
