// A set of matrices orthogonalised by Newton-Schulz products, the update direction of the Muon optimiser: with
// X = G / |G|_F (on the smaller side, m <= n) every step replaces the singular values s of X by p(s) = a s + b s^3 + c s^5,
//
//   A = X X^T;   B = b A + c A A;   X <- a X + B X        (m^2 n + m^3 + m^2 n multiply-adds)
//
// Arithmetic.  gfx950 multiplies fp32 matrices at 1/16 of its fp16 rate.  Every matrix here is bounded (the singular values
// stay below 2, so do all entries), so it is kept as two fp16 planes of the scaled value, hi = fp16(x S), lo = fp16(x S - hi),
// S = 2^13: 22 bits, with an absolute floor of 2^-38.  A product is three MFMAs, hi hi + hi lo + lo hi, accumulated in
// fp32; the dropped lo lo is 2^-22 relative, as the planes' own rounding.  That is fp32 accuracy at 1/3 of the fp16 rate.
// G is scaled by a power of two, exactly; the rest of the division by its norm (a factor r in (1, 2]) goes into the
// coefficients of the first step: a r, b r^3, c r^5.
//
// Layout.  A row of any matrix is a run of 128-byte blocks: 32 hi followed by 32 lo of the same columns, padded with zeros
// to whole tiles.  All three products contract over contiguous rows ("N T" form): X X^T and A A as they are (A is
// symmetric), B X against the rows of X^T, which is kept beside X: an output tile is written in both orientations.  The
// two symmetric products compute the tiles on and above the diagonal alone and write each also mirrored.
//
// Launches.  The matrices of a call go through each product together, one grid over all their tiles: an optimiser step on a
// model's many small matrices is 17 launches, whatever their number (up to 32 per group).
#include "common.h"
#include "dvae_hip.h"
#include "seq_common.h"
#include <math.h>

namespace dvae {

typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h16x4 __attribute__((ext_vector_type(4)));
typedef float nsf32x16 __attribute__((ext_vector_type(16)));
typedef unsigned nsu32x4 __attribute__((ext_vector_type(4)));

constexpr int NS_GROUP = 32;          // matrices per launch
constexpr int NS_PARTS = 64;          // partial sums of a norm
constexpr float NS_S = 8192.f;        // 2^13
constexpr int NS_LDS_ROW = 128 + 16;  // bytes: a 16-lane group's fragments fall on all banks

struct NsMat {
    const void* g;
    void* out;
    long ld_g, ld_out;
    long base;       // byte offset of its buffers: X, X^T, X', X'^T, A, B
    int rows, cols;  // of G
    int tile0;       // first tile of this launch
    __host__ __device__ int m() const { return rows < cols ? rows : cols; }
    __host__ __device__ int n() const { return rows < cols ? cols : rows; }
};
struct NsGroup {
    NsMat mat[NS_GROUP];
    int count, dtype;
    char* ws;
    double* parts;  // [count][NS_PARTS]
    float* r;       // [count]
    float a, b, c;
};

__host__ __device__ inline int ns_pad(int v, int tb) { return (v + tb - 1) / tb * tb; }
__host__ __device__ inline long ns_bytes(int mp, int np) { return (long)mp * np * 4; }
// 0 / 1: X / X^T, 2 / 3: the other pair, 4: A, 5: B
__host__ __device__ inline long ns_offset(int mp, int np, int which) {
    const long x = ns_bytes(mp, np);
    return which < 4 ? which * x : 4 * x + (which - 4) * ns_bytes(mp, mp);
}
// byte of column k in a row of blocks, plane 0 (hi); plane 1 is 64 bytes behind
__device__ __forceinline__ int ns_col(int k) { return (k >> 5) * 128 + (k & 31) * 2; }

// which matrix a unit of the grid belongs to
__device__ __forceinline__ int ns_find(const NsGroup& p, int unit) {
    int k = 0;
    while (k + 1 < p.count && unit >= p.mat[k + 1].tile0) ++k;
    return k;
}

template <typename T> __device__ __forceinline__ void ns_sum(const NsMat& m, double* out) {
    const T* g = (const T*)m.g;
    double s = 0;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < (long)m.rows * m.cols; i += NS_PARTS * 256) {
        const double v = (double)(float)g[(i / m.cols) * m.ld_g + i % m.cols];
        s += v * v;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    __shared__ double w[4];
    if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) *out = w[0] + w[1] + w[2] + w[3];
}
// |G|_F^2 in 64 bits: no range of G overflows or vanishes
__global__ __launch_bounds__(256) void ns_norm_kernel(NsGroup p) {
    const NsMat& m = p.mat[blockIdx.y];
    double* out = p.parts + blockIdx.y * NS_PARTS + blockIdx.x;
    if (p.dtype == DVAE_F32) ns_sum<float>(m, out);
    else if (p.dtype == DVAE_BF16) ns_sum<__bf16>(m, out);
    else ns_sum<_Float16>(m, out);
}

__device__ __forceinline__ void ns_split(float v, _Float16& hi, _Float16& lo) {
    hi = (_Float16)v;
    lo = (_Float16)(v - (float)hi);
}

// G -> X and X^T in planes: 64 x 64 tiles of G (padding included) through LDS
__global__ __launch_bounds__(256) void ns_split_kernel(NsGroup p, int tb) {
    __shared__ float tile[64][65];
    __shared__ int expo;
    const int k = ns_find(p, blockIdx.x);
    const NsMat& m = p.mat[k];
    const int rp = ns_pad(m.rows, tb), cp = ns_pad(m.cols, tb);
    const int t = blockIdx.x - m.tile0, r0 = t / (cp / 64) * 64, c0 = t % (cp / 64) * 64;
    if (threadIdx.x < 64) {
        double s = p.parts[k * NS_PARTS + threadIdx.x];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
        if (threadIdx.x == 0) {
            int e = 0;
            const double f = frexp(sqrt(s), &e);  // |G| = f 2^e, f in [1/2, 1)
            expo = s > 0 && s < INFINITY ? e : 0;
            if (t == 0) p.r[k] = s > 0 ? (s < INFINITY ? (float)(1.0 / f) : NAN) : s == 0 ? 1.f : NAN;
        }
    }
    __syncthreads();
    const double scale = ldexp((double)NS_S, -expo);
    const int j = threadIdx.x & 63;
    for (int i = threadIdx.x >> 6; i < 64; i += 4) {
        float v = 0.f;
        if (r0 + i < m.rows && c0 + j < m.cols) {
            const long at = (long)(r0 + i) * m.ld_g + c0 + j;
            v = p.dtype == DVAE_F32 ? ((const float*)m.g)[at] : p.dtype == DVAE_BF16 ? (float)((const __bf16*)m.g)[at] : (float)((const _Float16*)m.g)[at];
            v = (float)((double)v * scale);
        }
        tile[i][j] = v;
    }
    __syncthreads();
    const bool wide = m.rows <= m.cols;
    const int mp = wide ? rp : cp, np = wide ? cp : rp;
    char* straight = p.ws + m.base + ns_offset(mp, np, wide ? 0 : 1);  // rows as G's
    char* turned = p.ws + m.base + ns_offset(mp, np, wide ? 1 : 0);
    for (int i = threadIdx.x >> 6; i < 64; i += 4) {
        _Float16 hi, lo;
        ns_split(tile[i][j], hi, lo);
        char* at = straight + (long)(r0 + i) * cp * 4 + ns_col(c0 + j);
        *(_Float16*)at = hi;
        *(_Float16*)(at + 64) = lo;
        ns_split(tile[j][i], hi, lo);
        at = turned + (long)(c0 + i) * rp * 4 + ns_col(r0 + j);
        *(_Float16*)at = hi;
        *(_Float16*)(at + 64) = lo;
    }
}

enum { NS_GRAM, NS_POLY, NS_STEP, NS_LAST };

// One of the products, TB x TB output tiles, 4 waves as 2 x 2, each TB/2 x TB/2 of 32 x 32 MFMA blocks.  A stage of the K
// loop is one block (32 columns, both planes) of TB rows of either operand; the next stage's loads are in flight during
// the MFMAs and go to the other half of LDS behind them.
template <int TB, int MODE>
__global__ __launch_bounds__(256) void ns_product_kernel(NsGroup p, int from, int first) {
    constexpr int TM = TB / 64;
    constexpr int PASSES = TB / 32;  // 16 bytes per thread and pass: 32 rows
    constexpr int OPERAND = TB * NS_LDS_ROW;
    __shared__ __attribute__((aligned(16))) char lds[2][2 * OPERAND];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // workgroups that share an XCD (equal id mod 8) take neighbouring tiles
    const int q = gridDim.x >> 3, rest = gridDim.x & 7, xcd = blockIdx.x & 7;
    const int unit = (xcd < rest ? xcd * (q + 1) : rest * (q + 1) + (xcd - rest) * q) + (blockIdx.x >> 3);
    const int k = ns_find(p, unit);
    const NsMat& m = p.mat[k];
    const int mp = ns_pad(m.m(), TB), np = ns_pad(m.n(), TB), mt = mp / TB, nt = np / TB;
    const int t = unit - m.tile0;
    int ti, tj;
    if (MODE == NS_GRAM || MODE == NS_POLY) {  // row by row of the upper triangle: row i begins at i mt - i (i - 1) / 2
        ti = (int)((2 * mt + 1 - sqrtf((float)((2 * mt + 1) * (2 * mt + 1) - 8 * t))) * 0.5f);
        while (ti > 0 && ti * mt - ti * (ti - 1) / 2 > t) --ti;
        while ((ti + 1) * mt - (ti + 1) * ti / 2 <= t) ++ti;
        tj = ti + t - (ti * mt - ti * (ti - 1) / 2);
    } else {  // bands of 8 tile rows, column by column
        const int band = t / (8 * nt), in = t % (8 * nt), rows = min(8, mt - band * 8);
        ti = band * 8 + in % rows;
        tj = in / rows;
    }
    char* const base = p.ws + m.base;
    const long pitch = (long)(MODE == NS_GRAM ? np : mp) * 4;  // of both operands
    const char* a_rows = base + ns_offset(mp, np, MODE == NS_GRAM ? from : MODE == NS_POLY ? 4 : 5) + (long)ti * TB * pitch;
    const char* b_rows = base + ns_offset(mp, np, MODE == NS_GRAM ? from : MODE == NS_POLY ? 4 : from + 1) + (long)tj * TB * pitch;
    const int blocks = (int)(pitch / 128);

    nsf32x16 acc[TM][TM];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    const int wm = wave >> 1, wn = wave & 1;
    const long my = (long)(tid >> 3) * pitch + (tid & 7) * 16;
    const int my_lds = (tid >> 3) * NS_LDS_ROW + (tid & 7) * 16;
    nsu32x4 ra[PASSES], rb[PASSES];
    auto load = [&](int s) {
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            ra[i] = *(const nsu32x4*)(a_rows + my + i * 32 * pitch + (long)s * 128);
            rb[i] = *(const nsu32x4*)(b_rows + my + i * 32 * pitch + (long)s * 128);
        }
    };
    auto store = [&](char* l) {
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            *(nsu32x4*)(l + my_lds + i * 32 * NS_LDS_ROW) = ra[i];
            *(nsu32x4*)(l + OPERAND + my_lds + i * 32 * NS_LDS_ROW) = rb[i];
        }
    };
    load(0);
    store(lds[0]);
    load(min(1, blocks - 1));
    __syncthreads();
    // lane l of a fragment: row l & 31, columns 8 (l >> 5) .. + 7 of 16
    const int frag = (lane & 31) * NS_LDS_ROW + (lane >> 5) * 16;
    for (int s = 0; s < blocks; ++s) {
        const char* la = lds[s & 1] + wm * (TB / 2) * NS_LDS_ROW + frag;
        const char* lb = lds[s & 1] + OPERAND + wn * (TB / 2) * NS_LDS_ROW + frag;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            h16x8 ah[TM], al[TM], bh[TM], bl[TM];
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                ah[i] = *(const h16x8*)(la + i * 32 * NS_LDS_ROW + h * 32);
                al[i] = *(const h16x8*)(la + i * 32 * NS_LDS_ROW + h * 32 + 64);
                bh[i] = *(const h16x8*)(lb + i * 32 * NS_LDS_ROW + h * 32);
                bl[i] = *(const h16x8*)(lb + i * 32 * NS_LDS_ROW + h * 32 + 64);
            }
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TM; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al[i], bh[j], acc[i][j], 0, 0, 0);
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TM; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[i], bl[j], acc[i][j], 0, 0, 0);
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TM; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[i], bh[j], acc[i][j], 0, 0, 0);
            if (h == 0) {
                store(lds[(s & 1) ^ 1]);
                __builtin_amdgcn_sched_barrier(0);
                load(min(s + 2, blocks - 1));
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        __syncthreads();
    }

    // Epilogue.  Lane l of a block holds column l & 31 and rows (r & 3) + 8 (r >> 2) + 4 (l >> 5): quads of rows of one
    // column, which are contiguous in the turned copy.  The source of the added multiple is read from there.
    const float r = first ? p.r[k] : 1.f;
    const float unscale = 1.f / (NS_S * NS_S);
    const float from_src = MODE == NS_GRAM ? 0.f : MODE == NS_POLY ? p.b * r * r * r : p.a * r;
    const float from_acc = unscale * (MODE == NS_POLY ? p.c * r * r * r * r * r : 1.f);
    const char* src = base + ns_offset(mp, np, MODE == NS_POLY ? 4 : from + 1);  // rows of mp columns
    const int to = from ^ 2;
    char* straight = base + ns_offset(mp, np, MODE == NS_GRAM ? 4 : MODE == NS_POLY ? 5 : to);
    char* turned = MODE == NS_STEP ? base + ns_offset(mp, np, to + 1) : straight;
    const long straight_pitch = (long)(MODE == NS_STEP ? np : mp) * 4, turned_pitch = (long)mp * 4;
    const bool mirror = MODE == NS_STEP || ti != tj;  // a diagonal tile of a symmetric product has its mirror in itself
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) {
            const int col = tj * TB + wn * (TB / 2) + j * 32 + (lane & 31);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int row = ti * TB + wm * (TB / 2) + i * 32 + u * 8 + 4 * (lane >> 5);
                const long at = col * turned_pitch + ns_col(row);
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = acc[i][j][u * 4 + e] * from_acc;
                if (MODE != NS_GRAM) {
                    const h16x4 sh = *(const h16x4*)(src + at), sl = *(const h16x4*)(src + at + 64);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = fmaf(((float)sh[e] + (float)sl[e]) * (1.f / NS_S), from_src, v[e]);
                }
                if (MODE == NS_LAST) {
                    const bool wide = m.rows <= m.cols;
                    if (col >= m.n()) continue;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (row + e >= m.m()) continue;
                        const long o = wide ? (long)(row + e) * m.ld_out + col : (long)col * m.ld_out + row + e;
                        if (p.dtype == DVAE_F32) ((float*)m.out)[o] = v[e];
                        else if (p.dtype == DVAE_BF16) ((__bf16*)m.out)[o] = (__bf16)v[e];
                        else ((_Float16*)m.out)[o] = (_Float16)v[e];
                    }
                } else {
                    h16x4 hi, lo;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        _Float16 a, b;
                        ns_split(v[e] * NS_S, a, b);
                        hi[e] = a;
                        lo[e] = b;
                        char* o = straight + (row + e) * straight_pitch + ns_col(col);
                        *(_Float16*)o = a;
                        *(_Float16*)(o + 64) = b;
                    }
                    if (mirror) {
                        *(h16x4*)(turned + at) = hi;
                        *(h16x4*)(turned + at + 64) = lo;
                    }
                }
            }
        }
}

static int ns_cus() {
    static const int cus = [] {
        int dev = 0, n = 0;
        if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
        return n;
    }();
    return cus;
}

// tile of a call: 128 where the update products of a group fill the chip with them
static int ns_tile(const dvae_matrix_desc* d, int32_t count) {
    long tiles = 0;
    for (int i = 0; i < count; ++i) tiles += (long)cdiv(d[i].rows, 128) * cdiv(d[i].cols, 128);
    return tiles >= ns_cus() ? 128 : 64;
}
static long ns_matrix_bytes(const dvae_matrix_desc& d, int tb) {
    const int mp = ns_pad(d.rows < d.cols ? d.rows : d.cols, tb), np = ns_pad(d.rows < d.cols ? d.cols : d.rows, tb);
    return ns_offset(mp, np, 6);
}
constexpr long NS_HEAD = NS_GROUP * (NS_PARTS * 8 + 8);

static int ns_check(const char* who, const dvae_matrix_desc* d, int32_t count) {
    DVAE_REQUIRE(count >= 0 && (count == 0 || d), "%s: null pointer", who);
    for (int i = 0; i < count; ++i)
        DVAE_REQUIRE(d[i].rows >= 1 && d[i].cols >= 1 && d[i].rows <= 32768 && d[i].cols <= 32768,
                     "%s: matrix %d is %d x %d; sides of 1 .. 32768 are supported", who, i, d[i].rows, d[i].cols);
    return DVAE_OK;
}

}  // namespace dvae

extern "C" int64_t dvae_orthogonalize_ws_bytes(const dvae_matrix_desc* mats, int32_t count) {
    using namespace dvae;
    DVAE_TRY(ns_check("orthogonalize_ws_bytes", mats, count));
    int64_t most = 0;
    for (int g0 = 0; g0 < count; g0 += NS_GROUP) {  // the groups follow each other on the stream and share the space
        const int n = count - g0 < NS_GROUP ? count - g0 : NS_GROUP, tb = ns_tile(mats + g0, n);
        int64_t sum = NS_HEAD;
        for (int i = 0; i < n; ++i) sum += ns_matrix_bytes(mats[g0 + i], tb);
        most = sum > most ? sum : most;
    }
    return most;
}

extern "C" int dvae_orthogonalize(const dvae_matrix_desc* mats, int32_t count, int32_t steps, const float* coefficients,
                                  void* ws, int32_t dtype, void* stream) {
    using namespace dvae;
    DVAE_TRY(ns_check("orthogonalize", mats, count));
    DVAE_REQUIRE(known_dtype(dtype), "orthogonalize: unknown element type %d", dtype);
    DVAE_REQUIRE(steps >= 1 && steps <= 32 && coefficients, "orthogonalize: %d steps are not in 1 .. 32", steps);
    for (int i = 0; i < count; ++i)
        DVAE_REQUIRE(mats[i].g && mats[i].out && mats[i].ld_g >= mats[i].cols && mats[i].ld_out >= mats[i].cols,
                     "orthogonalize: matrix %d has a null pointer or a row stride below its columns", i);
    {  // the planes hold |X| <= 2, |A| <= 4, |B| < 8: follow the singular values through the steps
        constexpr int GRID = 4096;
        static thread_local float sigma[GRID + 1];
        for (int i = 0; i <= GRID; ++i) sigma[i] = (float)i / GRID;
        for (int t = 0; t < steps; ++t) {
            const float a = coefficients[3 * t], b = coefficients[3 * t + 1], c = coefficients[3 * t + 2];
            for (int i = 0; i <= GRID; ++i) {
                const float l = sigma[i] * sigma[i], poly = b * l + c * l * l;
                sigma[i] = (a + poly) * sigma[i];
                // (the first step's B carries r <= 2)
                DVAE_REQUIRE(fabsf(poly) * (t == 0 ? 2.f : 1.f) < 7.5f && fabsf(sigma[i]) < 1.95f,
                             "orthogonalize: with the coefficients of step %d singular values leave [-2, 2]", t);
            }
        }
    }
    if (count == 0) return DVAE_OK;
    DVAE_REQUIRE(ws && (uintptr_t)ws % 16 == 0, "orthogonalize: the workspace must be 16-byte aligned");
    hipStream_t s = (hipStream_t)stream;
    for (int g0 = 0; g0 < count; g0 += NS_GROUP) {
        const int n = count - g0 < NS_GROUP ? count - g0 : NS_GROUP, tb = ns_tile(mats + g0, n);
        NsGroup p = {};
        p.count = n;
        p.dtype = dtype;
        p.parts = (double*)ws;
        p.r = (float*)((char*)ws + NS_GROUP * NS_PARTS * 8);
        p.ws = (char*)ws + NS_HEAD;
        long base = 0;
        int split = 0, square = 0, update = 0;
        int tri0[NS_GROUP], upd0[NS_GROUP], spl0[NS_GROUP];
        for (int i = 0; i < n; ++i) {
            const dvae_matrix_desc& d = mats[g0 + i];
            NsMat& m = p.mat[i];
            m.g = d.g; m.out = d.out; m.ld_g = d.ld_g; m.ld_out = d.ld_out; m.rows = d.rows; m.cols = d.cols; m.base = base;
            base += ns_matrix_bytes(d, tb);
            const int mt = ns_pad(m.m(), tb) / tb, nt = ns_pad(m.n(), tb) / tb;
            spl0[i] = split; tri0[i] = square; upd0[i] = update;
            split += mt * nt * (tb / 64) * (tb / 64);
            square += mt * (mt + 1) / 2;
            update += mt * nt;
        }
        auto place = [&](const int* at) { for (int i = 0; i < n; ++i) p.mat[i].tile0 = at[i]; };
        hipLaunchKernelGGL(ns_norm_kernel, dim3(NS_PARTS, n), dim3(256), 0, s, p);
        DVAE_LAUNCH_CHECK();
        place(spl0);
        hipLaunchKernelGGL(ns_split_kernel, dim3(split), dim3(256), 0, s, p, tb);
        DVAE_LAUNCH_CHECK();
#define NS_PRODUCT(MODE, grid)                                                                                                 \
    do {                                                                                                                       \
        if (tb == 128) hipLaunchKernelGGL((ns_product_kernel<128, MODE>), dim3(grid), dim3(256), 0, s, p, 2 * (t & 1), t == 0); \
        else hipLaunchKernelGGL((ns_product_kernel<64, MODE>), dim3(grid), dim3(256), 0, s, p, 2 * (t & 1), t == 0);           \
        DVAE_LAUNCH_CHECK();                                                                                                   \
    } while (0)
        for (int t = 0; t < steps; ++t) {
            p.a = coefficients[3 * t]; p.b = coefficients[3 * t + 1]; p.c = coefficients[3 * t + 2];
            place(tri0);
            NS_PRODUCT(NS_GRAM, square);
            NS_PRODUCT(NS_POLY, square);
            place(upd0);
            if (t + 1 < steps) NS_PRODUCT(NS_STEP, update);
            else NS_PRODUCT(NS_LAST, update);
        }
#undef NS_PRODUCT
    }
    return DVAE_OK;
}
