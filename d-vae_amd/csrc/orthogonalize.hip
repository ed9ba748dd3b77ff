// A set of matrices orthogonalised by Newton-Schulz products, the update direction of the Muon optimiser: with
// X = G / |G|_F (on the smaller side, m <= n) every step replaces the singular values s of X by p(s) = a s + b s^3 + c s^5,
//
//   A = X X^T;   B = b A + c A A;   X <- a X + B X        (m^2 n + m^3 + m^2 n multiply-adds)
//
// Arithmetic.  gfx950 multiplies fp32 matrices at 1/16 of its fp16 rate.  Every matrix here is bounded (the singular values
// stay below 2, so do all entries), so it is kept as two fp16 planes of the scaled value, hi = fp16(x S), lo = fp16(x S - hi),
// S = 2^13: 22 bits, with an absolute floor of 2^-38.  A product is three MFMAs, hi hi + hi lo + lo hi, accumulated in
// fp32; the dropped lo lo is 2^-22 relative, as the planes' own rounding.  That is fp32 accuracy at 1/3 of the fp16 rate:
// against 64 bits the result is 7e-7 off at 501 x 501 and 3e-6 at 4096 x 4096, where the same iteration in fp32 is 2.2e-6 and 5e-6.
// With few rows the roundings average out less.  So
//   - up to 64 rows, and wherever the direct kernel runs, lo lo is added (latency bounds those products and hides it);
//   - up to 64 rows B is kept as B + f, f = -(b + c), with X <- (a - f) X + (B + f) X: where the singular values have come near 1, B
//     is near -f, and its rounding and the cancellation with a X are what is left (with many rows, small singular values leave
//     entries near 0 in B, which a shift would round worse);
//   - the sums of X X^T, over whole rows of X, are held in parts on 64 x 64 tiles and in the direct kernel: the products with a
//     second plane apart, hi hi in two or eight (one by one in fp32 9 x 1883 beside larger matrices was 2.7e-6 off and 9 x 20000
//     8.5e-6, where the fp32 iteration is 1.1e-6 and 3.5e-6; now 1.1e-6 and 0.9e-6; no time, the MFMAs are as many), and matrices
//     of up to 384 rows take 64 x 64 tiles there also in sets whose others take larger ones (five launches more: 60 us of 1400
//     with two 2048 x 2048 and three of few rows).
// Against the fp32 iteration's own error over random shapes and sets: median 0.9 of it up to 20 rows, 0.7 up to 65, 0.6 up to 400.
// G is scaled by a power of two, exactly; the rest of the division by its norm (a factor r in (1, 2]) goes into the
// coefficients of the first step: a r, b r^3, c r^5.
//
// Half products, where the caller asks for them (DVAE_HALF_PRODUCTS) and a bf16 matrix has sides of at least 512: the hi planes
// alone, one MFMA instead of three.  A, B and the operands X are then rounded to 11 bits; X itself keeps its second plane, which
// takes part in a X.  That is what matters: where a few singular values are far above the rest, as in gradients, the rounding of
// X would bury the small ones, which reach the result through a X (B is small there), while the same rounding inside a product
// meets the large directions only.  Measured against 64 bits, at 4096 x 4096 with four directions 0, 30 and 300 times the noise:
// 2.0e-3, 1.7e-3 and 1.6e-3, of which the result's own rounding to bf16 is 1.7e-3 (without X's second plane 1.9e-3, 8.7e-3 and
// 3.7e-2; the iteration in bf16 1.8e-2, 0.19 and 0.8).  Where many singular values end near each other it loses more: 2.5e-3 at
// 512 x 512 with equal ones.  A call takes 1490 us where full products take 3640 (1024 x 1024: 152 and 212).  Below 512 the roundings no longer average out (5e-3 at 9 x 1), so smaller matrices keep both planes;
// the choice looks at each matrix alone, and matrices of one and of two planes are launched apart.
//
// Layout.  A row of any matrix is a run of 128-byte blocks: 32 hi followed by 32 lo of the same columns, padded with zeros
// to whole tiles.  All three products contract over contiguous rows ("N T" form): X X^T and A A as they are (A is
// symmetric), B X against the rows of X^T, which is kept beside X: an output tile is written in both orientations.  The
// two symmetric products compute the tiles on and above the diagonal alone and write each also mirrored.
//
// Tiles.  The operands go straight from memory to LDS, several stages ahead.  Two things bound the products: what a CU can take
// in (17 to 21 bytes a cycle measured with all of them loading, whatever the depth; loads alone are 28 of the 29 us of the
// ENAS model's products X X^T and 35 of its update's 41), and with large tiles the power: the clock is 2.0 GHz where loads and
// MFMAs run together, 2.5 with either alone.  So a product takes the largest tile that still keeps the CUs busy:
//   256 x 256, one workgroup per CU, where the last round of them is nearly full: update at 4096 x 4096 350 to 370 us (1.1 to 1.2
//     PFLOP/s of MFMAs), half products 140 to 155 us (0.89 to 0.98 PFLOP/s; the epilogue is 40 us of either)
//   192 x 192 for symmetric products where their rounds cover less area than those of 128 x 128: 253 tiles are one round at
//     4096 x 4096 (185 to 215 us; half products 76 to 92), 528 of 128 x 128 two and a bit (half products 120 us)
//   128 x 128 from 3/4 of a tile per CU on (3000 x 3000: fp32 2600 -> 2220 us a call against 64 x 64, half products 1130 -> 990;
//     from 1/2 on the ENAS set would lose: 537 -> 677)
//   64 x 64; at most one per CU: four groups of waves share the sum (1024 x 1024: 242 us a call)
//   32 x 32, at most one per CU: the direct kernel (501 x 501: 155 -> 128 us a call; 768 x 768 would lose: 211 -> 232)
//
// Launches.  The matrices of a call go through each product together, one grid over all their tiles: an optimiser step on a
// model's many small matrices is 17 launches, whatever their number (up to 32 per group).  The coefficients are checked before
// the first of them in a few operations a step (0.5 us a call).
#include "common.h"
#include "dvae_hip.h"
#include "seq_common.h"
#include <math.h>

namespace dvae {

typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h16x4 __attribute__((ext_vector_type(4)));
typedef float nsf32x16 __attribute__((ext_vector_type(16)));
typedef float nsf32x4 __attribute__((ext_vector_type(4)));

constexpr int NS_GROUP = 32;          // matrices per launch
constexpr int NS_FEW = 384;           // rows up to which the long sums of X X^T are held apart; see the head of the file
constexpr int NS_PARTS = 256;         // partial sums of a norm
constexpr float NS_S = 8192.f;        // 2^13

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
    int count, dtype, planes, pad;  // sides are padded to whole multiples of `pad` with zeros
    char* ws;
    double* parts;  // [count][NS_PARTS]
    float* r;       // [count]
    float a, b, c, shift;  // of the step; what B of matrices with few rows is shifted by
};

__host__ __device__ inline int ns_pad(int v, int tb) { return (v + tb - 1) / tb * tb; }
__host__ __device__ inline long ns_bytes(int mp, int np, int planes) { return (long)mp * np * 2 * planes; }
// 0 / 1: X / X^T, 2 / 3: the other pair, 4: A, 5: B; with one plane also 6, 7: the second plane of X in either pair
__host__ __device__ inline long ns_offset(int mp, int np, int planes, int which) {
    const long x = ns_bytes(mp, np, planes), a = ns_bytes(mp, mp, planes);
    return which < 4 ? which * x : which < 6 ? 4 * x + (which - 4) * a : (which - 2) * x + 2 * a;
}
// byte of column k in a row of blocks; the second plane is 64 bytes behind
template <int PL> __device__ __forceinline__ int ns_col(int k) { return PL == 2 ? (k >> 5) * 128 + (k & 31) * 2 : k * 2; }

// which matrix a unit of the grid belongs to
__device__ __forceinline__ int ns_find(const NsGroup& p, int unit) {
    int k = 0;
    while (k + 1 < p.count && unit >= p.mat[k + 1].tile0) ++k;
    return k;
}

template <typename T, int V> __device__ __forceinline__ void ns_sum(const NsMat& m, double* out) {
    typedef T vec __attribute__((ext_vector_type(V)));
    // NS_PARTS x 4 waves: as many rows each as there are, and where there are few, shares of the columns
    constexpr int WAVES = NS_PARTS * 4, STEP = 64 * V;
    const int across = m.rows >= WAVES ? 1 : WAVES / m.rows, down = WAVES / across;
    const int wave = blockIdx.x * 4 + (threadIdx.x >> 6), r0 = wave / across, c0 = wave % across * STEP + (threadIdx.x & 63) * V;
    double s = 0;
    if (r0 < down)
        for (int r = r0; r < m.rows; r += down) {
            const T* row = (const T*)m.g + r * m.ld_g;
            for (int c = c0; c < m.cols; c += 4 * across * STEP) {  // four loads under way
                vec v[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int at = c + u * across * STEP;
                    v[u] = at < m.cols ? *(const vec*)(row + at) : vec{};
                }
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int e = 0; e < V; ++e) s += (double)(float)v[u][e] * (double)(float)v[u][e];
            }
        }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    __shared__ double w[4];
    if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) *out = w[0] + w[1] + w[2] + w[3];
}
// 16 bytes a load where all rows allow it
template <typename T> __device__ __forceinline__ void ns_sum(const NsMat& m, double* out) {
    constexpr int V = 16 / sizeof(T);
    if (((size_t)m.g | m.ld_g * sizeof(T)) % 16 == 0 && m.cols % V == 0) ns_sum<T, V>(m, out);
    else ns_sum<T, 1>(m, out);
}
// |G|_F^2 in 64 bits: no range of G overflows or vanishes
__global__ __launch_bounds__(256) void ns_norm_kernel(NsGroup p) {
    const NsMat& m = p.mat[blockIdx.y];
    double* out = p.parts + blockIdx.y * NS_PARTS + blockIdx.x;
    if (p.dtype == DVAE_F32) ns_sum<float>(m, out);
    else if (p.dtype == DVAE_BF16) ns_sum<__bf16>(m, out);
    else ns_sum<_Float16>(m, out);
}

// Eight scaled values to eight columns of a row of blocks
// (PL = 1: the second plane to `lo_at`, if there is one)
template <int PL> __device__ __forceinline__ void ns_put8(char* at, const float (&v)[8], char* lo_at = nullptr) {
    h16x8 hi, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        hi[e] = (_Float16)v[e];
        lo[e] = (_Float16)(v[e] - (float)hi[e]);
    }
    *(h16x8*)at = hi;
    if (PL == 2) *(h16x8*)(at + 64) = lo;
    else if (lo_at) *(h16x8*)lo_at = lo;
}

// G -> X and X^T in planes: 64 x 64 tiles of G (padding included) through LDS
template <int PL> __global__ __launch_bounds__(256) void ns_split_kernel(NsGroup p) {
    __shared__ float tile[64][65];
    __shared__ int expo;
    const int k = ns_find(p, blockIdx.x);
    const NsMat& m = p.mat[k];
    const int rp = ns_pad(m.rows, p.pad), cp = ns_pad(m.cols, p.pad);
    const int t = blockIdx.x - m.tile0, r0 = t / (cp / 64) * 64, c0 = t % (cp / 64) * 64;
    const int j = threadIdx.x & 63, i0 = threadIdx.x >> 6;
    float g[16];
#pragma unroll
    for (int u = 0; u < 16; ++u) {
        const int r = r0 + i0 + 4 * u, c = c0 + j;
        const long at = (long)min(r, m.rows - 1) * m.ld_g + min(c, m.cols - 1);
        const float v = p.dtype == DVAE_F32 ? ((const float*)m.g)[at] : p.dtype == DVAE_BF16 ? (float)((const __bf16*)m.g)[at] : (float)((const _Float16*)m.g)[at];
        g[u] = r < m.rows && c < m.cols ? v : 0.f;
    }
    if (threadIdx.x < 64) {
        double s = 0;
#pragma unroll
        for (int u = 0; u < NS_PARTS / 64; ++u) s += p.parts[k * NS_PARTS + u * 64 + threadIdx.x];
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
#pragma unroll
    for (int u = 0; u < 16; ++u) tile[i0 + 4 * u][j] = (float)((double)g[u] * scale);
    __syncthreads();
    const bool wide = m.rows <= m.cols;
    const int mp = wide ? rp : cp, np = wide ? cp : rp;
    char* straight = p.ws + m.base + ns_offset(mp, np, PL, wide ? 0 : 1);  // rows as G's
    char* turned = p.ws + m.base + ns_offset(mp, np, PL, wide ? 1 : 0);
#pragma unroll
    for (int u = threadIdx.x; u < 512; u += 256) {
        const int row = u >> 3, c8 = (u & 7) * 8;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = tile[row][c8 + e];
        char* const lo = p.ws + m.base + ns_offset(mp, np, PL, 6);
        const long straight_at = (long)(r0 + row) * cp * 2 * PL + ns_col<PL>(c0 + c8), turned_at = (long)(c0 + row) * rp * 2 * PL + ns_col<PL>(r0 + c8);
        ns_put8<PL>(straight + straight_at, v, wide ? lo + straight_at : nullptr);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = tile[c8 + e][row];
        ns_put8<PL>(turned + turned_at, v, wide ? nullptr : lo + turned_at);
    }
}

enum { NS_GRAM, NS_POLY, NS_STEP, NS_LAST };

// Tile t of mt x nt: the two symmetric products have those on and above the diagonal, row by row (row i begins at
// i mt - i (i - 1) / 2); the others go through bands of 8 tile rows column by column.
template <int MODE> __device__ __forceinline__ void ns_tile_at(int t, int mt, int nt, int& ti, int& tj) {
    if (MODE == NS_GRAM || MODE == NS_POLY) {
        ti = (int)((2 * mt + 1 - sqrtf((float)((2 * mt + 1) * (2 * mt + 1) - 8 * t))) * 0.5f);
        while (ti > 0 && ti * mt - ti * (ti - 1) / 2 > t) --ti;
        while ((ti + 1) * mt - (ti + 1) * ti / 2 <= t) ++ti;
        tj = ti + t - (ti * mt - ti * (ti - 1) / 2);
    } else {
        const int band = t / (8 * nt), in = t % (8 * nt), rows = min(8, mt - band * 8);
        ti = band * 8 + in % rows;
        tj = in / rows;
    }
}

// 16 bytes per lane from memory to LDS, without a register in between: lane l's go to `lds` + 16 l.  Not the builtin: the
// compiler would have every read of LDS wait for all of these loads; here ns_wait counts them.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 is no register of the compiler's: that it is clobbered is said all the same
__device__ __forceinline__ void ns_load_lds(const char* from, unsigned lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 1\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(from) : "memory", "m0");
}
#pragma clang diagnostic pop
// all but the last N loads of this wave are done and its reads of LDS too; then the workgroup meets
template <int N> __device__ __forceinline__ void ns_wait() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory"); }

// eight neighbours of a row of the result, rounded to its type
__device__ __forceinline__ void ns_out8(const NsMat& m, int dtype, int row, int col, const float (&v)[8]) {
    if (row >= m.rows || col >= m.cols) return;
    const int n = min(8, m.cols - col);
    char* at = (char*)m.out + (row * m.ld_out + col) * (dtype == DVAE_F32 ? 4 : 2);
    const bool whole = n == 8 && (size_t)at % 16 == 0;
    if (dtype == DVAE_F32) {
        if (whole) {
#pragma unroll
            for (int h = 0; h < 2; ++h) *(nsf32x4*)(at + 16 * h) = nsf32x4{v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]};
        } else
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < n) ((float*)at)[e] = v[e];
        return;
    }
    h16x8 bits;
#pragma unroll
    for (int e = 0; e < 8; ++e) bits[e] = dtype == DVAE_BF16 ? __builtin_bit_cast(_Float16, (__bf16)v[e]) : (_Float16)v[e];
    if (whole) *(h16x8*)at = bits;
    else
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < n) ((_Float16*)at)[e] = bits[e];
}

// One of the products, TB x TB output tiles; KG groups of waves, each with every KG-th stage of the sum; a group is 2 x WN
// waves of TB/2 x TB/WN outputs, TM x TN MFMA blocks of 32 x 32.  A stage of the sum is one block (32 columns in two planes,
// 64 in one) of TB rows of either operand; NB stages have room in LDS, the loads of all but the current one are under way.
template <int TB, int WN, int KG, int PL, int NB, int MODE>
__global__ __launch_bounds__(128 * WN * KG) void ns_product_kernel(NsGroup p, int from, int first) {
    constexpr int TM = TB / 64, TN = TB / WN / 32, NT = 128 * WN;
    constexpr bool SUMS = TB == 64 && PL == 2 && MODE == NS_GRAM;  // three sums of an output instead of one
    constexpr int LR = NT / 8, PASSES = TB / LR;  // 16 bytes per thread and pass: LR rows of one block
    constexpr int OPERAND = TB * 128, LOADS = 2 * PASSES;
    constexpr int TP = TB + 4;                    // row pitch of the output in LDS, floats; 64 rows at a time
    // 192 does not divide the padded sides: the last tiles reach over them, read the last row instead and store nothing there
    constexpr bool OVER = TB == 192;
    static_assert(NB >= 2 && 64 * TP * 4 <= NB * 2 * OPERAND && LR % 16 == 0 && (KG == 1 || TM == 1) && (!OVER || MODE == NS_GRAM || MODE == NS_POLY), "");
    constexpr int STAGED = KG * NB * 2 * OPERAND, OUT = (TM > 1 ? 2 : 1) * 64 * TP * 4;  // bytes: KG x NB stages; two blocks of the output
    __shared__ __attribute__((aligned(128))) char lds[STAGED > OUT ? STAGED : OUT];
    const int group = __builtin_amdgcn_readfirstlane(threadIdx.x / NT), tid = threadIdx.x % NT;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int k = ns_find(p, blockIdx.x);
    const NsMat& m = p.mat[k];
    const int mp = ns_pad(m.m(), p.pad), np = ns_pad(m.n(), p.pad), mt = OVER ? (mp + TB - 1) / TB : mp / TB, nt = np / TB;
    // workgroups that share an XCD (equal id mod 8) take neighbouring tiles of a matrix
    const int tiles = MODE == NS_GRAM || MODE == NS_POLY ? mt * (mt + 1) / 2 : mt * nt;
    const int local = blockIdx.x - m.tile0, q = tiles >> 3, rest = tiles & 7, xcd = local & 7;
    const int t = (xcd < rest ? xcd * (q + 1) : rest * (q + 1) + (xcd - rest) * q) + (local >> 3);
    int ti, tj;
    ns_tile_at<MODE>(t, mt, nt, ti, tj);
    char* const base = p.ws + m.base;
    const long pitch = (long)(MODE == NS_GRAM ? np : mp) * 2 * PL;  // of both operands
    const char* a_rows = base + ns_offset(mp, np, PL, MODE == NS_GRAM ? from : MODE == NS_POLY ? 4 : 5) + (long)ti * TB * pitch;
    const char* b_rows = base + ns_offset(mp, np, PL, MODE == NS_GRAM ? from : MODE == NS_POLY ? 4 : from + 1) + (long)tj * TB * pitch;
    const int blocks = (int)(pitch / 128), stages = (blocks + KG - 1) / KG;

    const bool few = PL == 2 && m.m() <= 64;  // lo lo too, and B shifted
    const int col0 = tj * TB;
    const bool mirror = MODE == NS_STEP || ((MODE == NS_GRAM || MODE == NS_POLY) && ti != tj);  // a diagonal tile is its own mirror
    const char* src = base + ns_offset(mp, np, PL, MODE == NS_POLY ? 4 : from);
    char* dst = base + ns_offset(mp, np, PL, MODE == NS_GRAM ? 4 : MODE == NS_POLY ? 5 : from ^ 2);
    char* turned = base + ns_offset(mp, np, PL, MODE == NS_GRAM ? 4 : MODE == NS_POLY ? 5 : (from ^ 2) + 1);
    constexpr bool CARRY = PL == 1 && (MODE == NS_STEP || MODE == NS_LAST);  // X's second plane goes through the epilogue alone
    const char* src_lo_plane = base + ns_offset(mp, np, PL, 6 + from / 2);
    char* dst_lo = base + ns_offset(mp, np, PL, 6 + (from ^ 2) / 2);
    const long row_bytes = (long)(MODE == NS_STEP || MODE == NS_LAST ? np : mp) * 2 * PL;
    auto row_of = [&](int i, int row) { return ti * TB + (row >> 5) * (TB / 2) + i * 32 + (row & 31); };
    // The source of the added multiple for block row i, a thread's n-th eight values, is read ahead: for the first one from
    // the start (64 x 64) or during the last stage, for the others while the one before is written.
    constexpr int UNITS = (64 * TB / 8 + NT * KG - 1) / (NT * KG);
    constexpr bool FROM_START = TB == 64, FROM_LAST = !FROM_START && !(TB == 256 && PL == 2);  // (there no registers are left)
    h16x8 src_hi[UNITS], src_lo[UNITS];
    auto fetch = [&](int i, int n) {
        const int u = min((int)threadIdx.x + n * NT * KG, 64 * TB / 8 - 1), row = row_of(i, u / (TB / 8)), c = col0 + u % (TB / 8) * 8;
        const char* at = src + (long)(OVER ? min(row, mp - 1) : row) * row_bytes + ns_col<PL>(OVER ? min(c, mp - 8) : c);
        src_hi[n] = *(const h16x8*)at;
        if (PL == 2) src_lo[n] = *(const h16x8*)(at + 64);
        else if (CARRY) src_lo[n] = *(const h16x8*)(src_lo_plane + (at - src));
        else src_lo[n] = h16x8{};
    };
    if (MODE != NS_GRAM && FROM_START)
#pragma unroll
        for (int n = 0; n < UNITS; ++n) fetch(0, n);

    nsf32x16 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    nsf32x16 odd, cross;  // SUMS: of every other 16 columns, and of the products with a second plane
#pragma unroll
    for (int r = 0; r < 16; ++r) odd[r] = cross[r] = 0.f;
    const int wm = wave / WN, wn = wave % WN;
    // A wave's load writes 1 KB of LDS in the order of its lanes: 8 rows of 128 bytes.  Chunk c of row r goes to place
    // c ^ (r / 2 mod 8), so that the 16 rows that a read of a fragment takes at a time lie on different banks.
    const int chunk = (tid & 7) ^ (tid >> 4 & 7);
    int at_a[PASSES], at_b[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int row = (tid >> 3) + i * LR;
        at_a[i] = (OVER ? min(row, mp - 1 - ti * TB) : row) * (int)pitch + chunk * 16;
        at_b[i] = (OVER ? min(row, mp - 1 - tj * TB) : row) * (int)pitch + chunk * 16;
    }
    const unsigned lds0 = __builtin_amdgcn_readfirstlane((unsigned)(size_t)(__attribute__((address_space(3))) char*)(lds + group * NB * 2 * OPERAND + wave * 1024));
    // one of the loads of stage s, into buffer b; past the last block the last one is loaded again and not used
    auto load = [&](int b, int s, int n) {
        const long block = (long)min(s * KG + group, blocks - 1) * 128;
        if (n & 1) ns_load_lds(b_rows + block + at_b[n >> 1], lds0 + b * 2 * OPERAND + OPERAND + (n >> 1) * LR * 128);
        else ns_load_lds(a_rows + block + at_a[n >> 1], lds0 + b * 2 * OPERAND + (n >> 1) * LR * 128);
    };
    // lane l of a fragment: row l & 31, columns 8 (l >> 5) .. + 7 of 16
    constexpr int SUB = PL == 2 ? 2 : 4;  // 16-column steps of a stage
    const int swizzle = lane >> 1 & 7;
    int frag[4];  // chunk 2 n + (l >> 5) of the lane's row
#pragma unroll
    for (int n = 0; n < 4; ++n) frag[n] = (lane & 31) * 128 + ((2 * n + (lane >> 5)) ^ swizzle) * 16;
    // PIPED: a fragment is read while the one before is multiplied, and a stage's loads are issued among the products: all
    // at once they would hold up the wave until the memory path has taken them.  Two workgroups per CU do that for each other.
    constexpr bool PIPED = TB != 128 && KG == 1 && !(TB == 256 && PL == 2);  // (nor are there registers for it in the latter)
    h16x8 fa[2][PL][TM], fb[2][PL][TN];
    auto read = [&](int to, int b, int h) {
        const char* la = (char*)lds + (group * NB + b) * 2 * OPERAND + wm * (TB / 2) * 128;
        const char* lb = (char*)lds + (group * NB + b) * 2 * OPERAND + OPERAND + wn * (TB / WN) * 128;
#pragma unroll
        for (int q = 0; q < PL; ++q) {
#pragma unroll
            for (int i = 0; i < TM; ++i) fa[to][q][i] = *(const h16x8*)(la + i * 32 * 128 + frag[h + 2 * q]);
#pragma unroll
            for (int j = 0; j < TN; ++j) fb[to][q][j] = *(const h16x8*)(lb + j * 32 * 128 + frag[h + 2 * q]);
        }
    };
    auto arrive = [&](int s) {  // the loads of stage s are done, everywhere; all fragments asked for so far are read
        if (NB > 2 && s + NB - 2 < stages) ns_wait<(NB - 2) * LOADS>();
        else ns_wait<0>();
    };
#pragma unroll
    for (int s = 0; s < NB - 1; ++s)
        if (s < stages)
#pragma unroll
            for (int n = 0; n < LOADS; ++n) load(s, s, n);
    if (PIPED) {
        arrive(0);
        read(0, 0, 0);
    }
    int b = 0;
    for (int s = 0; s < stages; ++s) {
        const int after = b + 1 == NB ? 0 : b + 1, before = b == 0 ? NB - 1 : b - 1;
        const bool mine = KG == 1 || s * KG + group < blocks, more = s + NB - 1 < stages;
        constexpr int PRODUCTS = PL == 2 ? 3 : 1, GROUPS = (SUB - 1) * PRODUCTS * TM, EACH = (LOADS + GROUPS - 1) / GROUPS;
        if (!PIPED) {
            arrive(s);
            if (more)
#pragma unroll
                for (int n = 0; n < LOADS; ++n) load(before, s + NB - 1, n);
        }
        if (MODE != NS_GRAM && FROM_LAST && s + 1 == stages)
#pragma unroll
            for (int n = 0; n < UNITS; ++n) fetch(0, n);
        int n = 0;
#pragma unroll
        for (int h = 0; h < SUB; ++h) {
            if (!PIPED) read(h & 1, b, h);
            else if (h + 1 < SUB) read((h + 1) & 1, b, h + 1);
            else if (s + 1 < stages) {
                arrive(s + 1);
                read(0, after, 0);
            }
            if (PIPED) __builtin_amdgcn_sched_barrier(0);
            auto mma = [&](int qa, int qb, int i) {
#pragma unroll
                for (int j = 0; j < TN; ++j) {
                    nsf32x16& sum = SUMS && qa + qb > 0 ? cross : SUMS && (h & 1) ? odd : acc[i][j];
                    sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[h & 1][qa][i], fb[h & 1][qb][j], sum, 0, 0, 0);
                }
            };
#pragma unroll
            for (int q = 0; q < PRODUCTS; ++q)
#pragma unroll
                for (int i = 0; i < TM; ++i) {
                    if (mine) {
                        if (PL == 2 && q == 0 && few) mma(PL - 1, PL - 1, i);
                        mma(PL == 2 && q == 0, PL == 2 && q == 1, i);
                    }
                    if (PIPED) {
                        if (h + 1 < SUB)
#pragma unroll
                            for (int u = 0; u < EACH; ++u, ++n)
                                if (n < LOADS && more) load(before, s + NB - 1, n);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
        }
        b = after;
    }
    if (SUMS) acc[0][0] += odd + cross;
    if (MODE != NS_GRAM && !FROM_START && !FROM_LAST)
#pragma unroll
        for (int n = 0; n < UNITS; ++n) fetch(0, n);
    __syncthreads();

    // Epilogue: the output goes through LDS, one 32-row block of either wave row at a time, so that every access to memory
    // is 16 bytes of a row in either orientation; the groups' sums meet there, in their order.  Column c of row q stands at
    // c ^ 8 (q / 8 mod 8): rows are read 8 columns at a time and columns 8 rows at a time, both from all banks.
    // Lane l of an MFMA block holds column l & 31 and rows (r & 3) + 8 (r >> 2) + 4 (l >> 5).
    const float r = first ? p.r[k] : 1.f;
    const float shift = few ? p.shift : 0.f;
    const float from_src = MODE == NS_GRAM ? 0.f : (MODE == NS_POLY ? p.b * r * r * r : (p.a - shift) * r) / NS_S;
    const float from_acc = (MODE == NS_POLY ? p.c * r * r * r * r * r : 1.f) / (NS_S * NS_S);
    const bool wide = m.rows <= m.cols;  // else the rows of out are the columns of X
    auto place = [](int row, int c) { return row * TP + (c ^ (row & 56)); };
    constexpr int GROUP_FLOATS = NB * 2 * OPERAND / 4;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        float* const tile = (float*)lds + (i & 1) * 64 * TP;
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                tile[group * GROUP_FLOATS + place(wm * 32 + (e & 3) + 8 * (e >> 2) + 4 * (lane >> 5), wn * (TB / WN) + j * 32 + (lane & 31))] =
                    acc[i][j][e] * from_acc;
        __syncthreads();
#pragma unroll
        for (int n = 0; n < UNITS; ++n) {
            const int u = threadIdx.x + n * NT * KG, row = u / (TB / 8), c8 = u % (TB / 8) * 8;
            if (64 * TB / 8 % (NT * KG) && u >= 64 * TB / 8) break;
            if (OVER && (row_of(i, row) >= mp || col0 + c8 >= mp)) continue;
            const long at = (long)row_of(i, row) * row_bytes + ns_col<PL>(col0 + c8);
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = tile[place(row, c8) + e];
#pragma unroll
                for (int g = 1; g < KG; ++g) v[e] += tile[g * GROUP_FLOATS + place(row, c8) + e];
            }
            if (MODE != NS_GRAM) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = fmaf((float)src_hi[n][e] + (float)src_lo[n][e], from_src, v[e]);
                if (MODE == NS_POLY && few)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (row_of(i, row) == col0 + c8 + e) v[e] += shift * r;
                if (i + 1 < TM) fetch(i + 1, n);
            }
            if ((MODE != NS_GRAM || KG > 1) && (MODE == NS_LAST ? !wide : mirror))
#pragma unroll
                for (int e = 0; e < 8; ++e) tile[place(row, c8) + e] = v[e];
            if (MODE != NS_LAST) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] *= NS_S;
                ns_put8<PL>(dst + at, v, CARRY ? dst_lo + at : nullptr);
            } else if (wide) ns_out8(m, p.dtype, row_of(i, row), col0 + c8, v);
        }
        if (MODE == NS_LAST ? !wide : mirror) {
            if (MODE != NS_GRAM || KG > 1) __syncthreads();
#pragma unroll
            for (int n = 0; n < UNITS; ++n) {
                const int u = threadIdx.x + n * NT * KG, c = u / 8, r8 = u % 8 * 8;
                if (64 * TB / 8 % (NT * KG) && u >= 64 * TB / 8) break;
                if (OVER && (row_of(i, r8) >= mp || col0 + c >= mp)) continue;
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = tile[place(r8 + e, c)] * (MODE == NS_LAST ? 1.f : NS_S);
                if (MODE == NS_LAST) ns_out8(m, p.dtype, col0 + c, row_of(i, r8), v);
                else ns_put8<PL>(turned + (long)(col0 + c) * mp * 2 * PL + ns_col<PL>(row_of(i, r8)), v);
            }
        }
    }
}

// The same products where they are small and their latency counts: 32 x 32 output tiles, one MFMA block each, the eight waves
// of a workgroup take every eighth block of the sum.  Fragments come straight from memory (a lane's 16 bytes are 16 bytes of a
// row), two blocks in flight per wave; no LDS and no barrier until the waves' sums meet.
template <int PL, int MODE>
__global__ __launch_bounds__(512) void ns_small_kernel(NsGroup p, int from, int first) {
    constexpr int W = 8, TP = 36;
    __shared__ __attribute__((aligned(16))) float part[W][32 * TP];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int k = ns_find(p, blockIdx.x);
    const NsMat& m = p.mat[k];
    const int mp = ns_pad(m.m(), p.pad), np = ns_pad(m.n(), p.pad);
    int ti, tj;
    ns_tile_at<MODE>(blockIdx.x - m.tile0, mp / 32, np / 32, ti, tj);
    char* const base = p.ws + m.base;
    const long pitch = (long)(MODE == NS_GRAM ? np : mp) * 2 * PL;
    const char* a_rows = base + ns_offset(mp, np, PL, MODE == NS_GRAM ? from : MODE == NS_POLY ? 4 : 5);
    const char* b_rows = base + ns_offset(mp, np, PL, MODE == NS_GRAM ? from : MODE == NS_POLY ? 4 : from + 1);
    a_rows += (long)(ti * 32 + (lane & 31)) * pitch + (lane >> 5) * 16;
    b_rows += (long)(tj * 32 + (lane & 31)) * pitch + (lane >> 5) * 16;
    const int blocks = (int)(pitch / 128);
    // the source of the added multiple is under way from the start: thread u < 128 has row u / 4, columns 8 (u % 4) ..
    const int row = (threadIdx.x >> 2) & 31, c8 = (threadIdx.x & 3) * 8;
    const long row_bytes = (long)(MODE == NS_STEP || MODE == NS_LAST ? np : mp) * 2 * PL;
    const long at = (long)(ti * 32 + row) * row_bytes + ns_col<PL>(tj * 32 + c8);
    constexpr bool CARRY = PL == 1 && (MODE == NS_STEP || MODE == NS_LAST);
    h16x8 src_hi = {}, src_lo = {};
    if (MODE != NS_GRAM && threadIdx.x < 128) {
        const char* src = base + ns_offset(mp, np, PL, MODE == NS_POLY ? 4 : from) + at;
        src_hi = *(const h16x8*)src;
        if (PL == 2) src_lo = *(const h16x8*)(src + 64);
        if (CARRY) src_lo = *(const h16x8*)(base + ns_offset(mp, np, PL, 6 + from / 2) + at);
    }
    nsf32x16 acc, cross;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = cross[e] = 0.f;
    for (int s0 = wave; s0 < blocks; s0 += 2 * W) {
        h16x8 a[2][4], b[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int h = 0; h < 4; ++h) {  // two planes: hi hi lo lo; one plane: four 16-column steps
                const long o = (long)min(s0 + n * W, blocks - 1) * 128 + h * 32;
                a[n][h] = *(const h16x8*)(a_rows + o);
                b[n][h] = *(const h16x8*)(b_rows + o);
            }
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            if (s0 + n * W >= blocks) break;
            if (PL == 2) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[n][h + 2], b[n][h + 2], cross, 0, 0, 0);
                    cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[n][h + 2], b[n][h], cross, 0, 0, 0);
                    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[n][h], b[n][h], acc, 0, 0, 0);
                    cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[n][h], b[n][h + 2], cross, 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int h = 0; h < 4; ++h) acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[n][h], b[n][h], acc, 0, 0, 0);
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) part[wave][((e & 3) + 8 * (e >> 2) + 4 * (lane >> 5)) * TP + (lane & 31)] = acc[e] + cross[e];
    __syncthreads();
    const float r = first ? p.r[k] : 1.f, shift = PL == 2 && m.m() <= 64 ? p.shift : 0.f;
    const float from_src = MODE == NS_GRAM ? 0.f : (MODE == NS_POLY ? p.b * r * r * r : (p.a - shift) * r) / NS_S;
    const float from_acc = (MODE == NS_POLY ? p.c * r * r * r * r * r : 1.f) / (NS_S * NS_S);
    const bool mirror = MODE == NS_STEP || ((MODE == NS_GRAM || MODE == NS_POLY) && ti != tj);
    if (threadIdx.x < 128) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float t = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) t += part[w][row * TP + c8 + e];
            v[e] = fmaf((float)src_hi[e] + (float)src_lo[e], from_src, t * from_acc);
            if (MODE == NS_POLY && ti * 32 + row == tj * 32 + c8 + e) v[e] += shift * r;
            part[0][row * TP + c8 + e] = v[e];
        }
        if (MODE != NS_LAST) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= NS_S;
            ns_put8<PL>(base + ns_offset(mp, np, PL, MODE == NS_GRAM ? 4 : MODE == NS_POLY ? 5 : from ^ 2) + at, v,
                        CARRY ? base + ns_offset(mp, np, PL, 6 + (from ^ 2) / 2) + at : nullptr);
        }
    }
    __syncthreads();
    if (MODE == NS_LAST) {
        const bool wide = m.rows <= m.cols;
        for (int u = threadIdx.x; u < 1024; u += 512) {
            const int i = wide ? u >> 5 : u & 31, j = wide ? u & 31 : u >> 5, gr = ti * 32 + i, gc = tj * 32 + j;
            if (gr >= m.m() || gc >= m.n()) continue;
            const float v = part[0][i * TP + j];
            const long o = wide ? gr * m.ld_out + gc : gc * m.ld_out + gr;
            if (p.dtype == DVAE_F32) ((float*)m.out)[o] = v;
            else if (p.dtype == DVAE_BF16) ((__bf16*)m.out)[o] = (__bf16)v;
            else ((_Float16*)m.out)[o] = (_Float16)v;
        }
    } else if (mirror && threadIdx.x < 128) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = part[0][(c8 + e) * TP + row] * NS_S;  // here `row` is a column of the tile, c8 its rows
        ns_put8<PL>(base + ns_offset(mp, np, PL, MODE == NS_GRAM ? 4 : MODE == NS_POLY ? 5 : (from ^ 2) + 1) +
                        (long)(tj * 32 + row) * mp * 2 * PL + ns_col<PL>(ti * 32 + c8), v);
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

// A product runs on 128 x 128 tiles from 3/4 of one per CU on, else on 64 x 64.
static bool ns_big(long tiles128) { return 4 * tiles128 >= 3L * ns_cus(); }
// 256 x 256 tiles, one workgroup per CU, where the last round of them is nearly full.
static bool ns_huge(long tiles256) {
    const long rounds = (tiles256 + ns_cus() - 1) / ns_cus();
    return 8 * tiles256 >= 7 * rounds * ns_cus();
}
// what the sides are padded to: the largest tile that any product takes, where that adds at most an eighth to the work (eight
// 700 x 700: 449 us a call on 64 x 64, 514 on 128 x 128)
static int ns_pad_of(const dvae_matrix_desc* mats, const int* group, int n) {
    long small = 0, big = 0, huge = 0;
    for (int i = 0; i < n; ++i) {
        const dvae_matrix_desc& d = mats[group[i]];
        small += (long)cdiv(d.rows, 64) * cdiv(d.cols, 64);
        big += (long)cdiv(d.rows, 128) * cdiv(d.cols, 128);
        huge += (long)cdiv(d.rows, 256) * cdiv(d.cols, 256);
    }
    if (ns_huge(huge) && 32 * huge <= 9 * big) return 256;
    return ns_big(big) && 32 * big <= 9 * small ? 128 : 64;
}
static long ns_matrix_bytes(const dvae_matrix_desc& d, int pad, int planes) {
    const int mp = ns_pad(d.rows < d.cols ? d.rows : d.cols, pad), np = ns_pad(d.rows < d.cols ? d.cols : d.rows, pad);
    return ns_offset(mp, np, planes, planes == 1 ? 8 : 6);
}
// planes in the products of a matrix; see the head of the file
static int ns_planes(const dvae_matrix_desc& d, int half) { return half && d.rows >= 512 && d.cols >= 512 ? 1 : 2; }
// The call's matrices in groups that share their launches: up to NS_GROUP of the same number of planes, in the order of the call.
// First those of two planes; `at` and `planes` say where the next group begins.  Returns the group's size, 0 behind the last.
static int ns_next(const dvae_matrix_desc* d, int count, int half, int& planes, int& at, int (&group)[NS_GROUP]) {
    int n = 0;
    for (;; planes = 1, at = 0) {
        for (; at < count && n < NS_GROUP; ++at)
            if (ns_planes(d[at], half) == planes) group[n++] = at;
        if (n > 0 || planes == 1) return n;
    }
}
constexpr long NS_HEAD = NS_GROUP * (NS_PARTS * 8 + 8);

static int ns_check(const char* who, const dvae_matrix_desc* d, int32_t count, int32_t dtype) {
    DVAE_REQUIRE(known_dtype(dtype & ~DVAE_HALF_PRODUCTS), "%s: unknown element type %d", who, dtype);
    DVAE_REQUIRE(!(dtype & DVAE_HALF_PRODUCTS) || dtype == (DVAE_BF16 | DVAE_HALF_PRODUCTS), "%s: half products are for bf16 matrices", who);
    DVAE_REQUIRE(count >= 0 && (count == 0 || d), "%s: null pointer", who);
    for (int i = 0; i < count; ++i)
        DVAE_REQUIRE(d[i].rows >= 1 && d[i].cols >= 1 && d[i].rows <= 32768 && d[i].cols <= 32768,
                     "%s: matrix %d is %d x %d; sides of 1 .. 32768 are supported", who, i, d[i].rows, d[i].cols);
    return DVAE_OK;
}

}  // namespace dvae

extern "C" int64_t dvae_orthogonalize_ws_bytes(const dvae_matrix_desc* mats, int32_t count, int32_t dtype) {
    using namespace dvae;
    DVAE_TRY(ns_check("orthogonalize_ws_bytes", mats, count, dtype));
    int64_t most = 0;
    int group[NS_GROUP], planes = 2, at = 0;
    while (const int n = ns_next(mats, count, dtype & DVAE_HALF_PRODUCTS, planes, at, group)) {  // the groups follow each other on the stream and share the space
        const int pad = ns_pad_of(mats, group, n);
        int64_t sum = NS_HEAD;
        for (int i = 0; i < n; ++i) sum += ns_matrix_bytes(mats[group[i]], pad, planes);
        most = sum > most ? sum : most;
    }
    return most;
}

extern "C" int dvae_orthogonalize(const dvae_matrix_desc* mats, int32_t count, int32_t steps, const float* coefficients,
                                  void* ws, int32_t dtype, void* stream) {
    using namespace dvae;
    DVAE_TRY(ns_check("orthogonalize", mats, count, dtype));
    DVAE_REQUIRE(steps >= 1 && steps <= 32 && coefficients, "orthogonalize: %d steps are not in 1 .. 32", steps);
    for (int i = 0; i < count; ++i)
        DVAE_REQUIRE(mats[i].g && mats[i].out && mats[i].ld_g >= mats[i].cols && mats[i].ld_out >= mats[i].cols,
                     "orthogonalize: matrix %d has a null pointer or a row stride below its columns", i);
    // The planes hold |X| <= 2, |A| <= 4, |B| < 8.  The singular values of X fill at most [0, most], whose image under the odd
    // p(s) = a s + b s^3 + c s^5 is [0, max |p|] again in absolute values; with l = s^2 the maximum is at the end or where
    // a + 3 b l + 5 c l^2 = 0, that of B's |b l + c l^2| at the end or at l = -b / 2 c.
    double most = 1;
    float shift[32];
    for (int t = 0; t < steps; ++t) {
        const double a = coefficients[3 * t], b = coefficients[3 * t + 1], c = coefficients[3 * t + 2], end = most * most;
        auto p_at = [&](double l) { return fabs((a + b * l + c * l * l) * sqrt(l)); };
        auto b_at = [&](double l) { return b * l + c * l * l; };
        double low = fmin(0, b_at(end)), high = fmax(0, b_at(end));
        most = p_at(end);
        const double d = 9 * b * b - 20 * a * c;
        // (both roots of the quadratic without cancellation; infinite ones, as with c = 0, lie outside)
        const double q = d >= 0 ? -(3 * b + copysign(sqrt(d), b)) / 2 : 0, roots[3] = {q / (5 * c), a / q, -b / (2 * c)};
        for (int i = 0; i < 3; ++i) {
            if (!(roots[i] > 0 && roots[i] < end)) continue;
            if (i < 2) most = fmax(most, p_at(roots[i]));
            else low = fmin(low, b_at(roots[i])), high = fmax(high, b_at(roots[i]));
        }
        const double big = fmax(-low, high);
        DVAE_REQUIRE(most < 1.95, "orthogonalize: with the coefficients of step %d singular values leave [-2, 2]", t);
        // (the first step's B carries r <= 2)
        DVAE_REQUIRE(big * (t == 0 ? 2 : 1) < 7.5, "orthogonalize: the coefficients b and c of step %d are too large", t);
        shift[t] = (float)-(b + c);
        if (!(fmax(-(low + shift[t]), high + shift[t]) * (t == 0 ? 2 : 1) < 7.5)) shift[t] = 0;
    }
    if (count == 0) return DVAE_OK;
    DVAE_REQUIRE(ws && (uintptr_t)ws % 16 == 0, "orthogonalize: the workspace must be 16-byte aligned");
    hipStream_t s = (hipStream_t)stream;
    int order[NS_GROUP], planes = 2, next = 0;
    while (const int n = ns_next(mats, count, dtype & DVAE_HALF_PRODUCTS, planes, next, order)) {
        NsGroup p = {};
        p.count = n;
        p.dtype = dtype & ~DVAE_HALF_PRODUCTS;
        p.planes = planes;
        p.pad = ns_pad_of(mats, order, n);
        p.parts = (double*)ws;
        p.r = (float*)((char*)ws + NS_GROUP * NS_PARTS * 8);
        p.ws = (char*)ws + NS_HEAD;
        // the matrices with the longest sums first: their tiles are the last to end
        for (int i = 1; i < n; ++i)
            for (int j = i; j > 0; --j) {
                auto longer = [&](int k) { return mats[k].rows > mats[k].cols ? mats[k].rows : mats[k].cols; };
                if (longer(order[j]) <= longer(order[j - 1])) break;
                const int swap = order[j]; order[j] = order[j - 1]; order[j - 1] = swap;
            }
        long base = 0;
        int split = 0, square[5] = {}, update[5] = {};  // tiles of all matrices, of these sides:
        constexpr int side[5] = {32, 64, 128, 256, 192};
        int split0[NS_GROUP], square0[5][NS_GROUP], update0[5][NS_GROUP];
        for (int i = 0; i < n; ++i) {
            const dvae_matrix_desc& d = mats[order[i]];
            NsMat& m = p.mat[i];
            m.g = d.g; m.out = d.out; m.ld_g = d.ld_g; m.ld_out = d.ld_out; m.rows = d.rows; m.cols = d.cols; m.base = base;
            base += ns_matrix_bytes(d, p.pad, p.planes);
            const int mp = ns_pad(m.m(), p.pad), np = ns_pad(m.n(), p.pad);
            split0[i] = split;
            split += (mp / 64) * (np / 64);
            for (int b = 0; b < 5; ++b) {
                const int mt = cdiv(mp, side[b]), nt = cdiv(np, side[b]);
                square0[b][i] = square[b]; update0[b][i] = update[b];
                square[b] += mt * (mt + 1) / 2;
                update[b] += mt * nt;
            }
        }
        auto size = [&](const int* tiles) {
            return p.pad == 256 && ns_huge(tiles[3]) ? 3 : p.pad >= 128 && ns_big(tiles[2]) ? 2 : tiles[0] <= ns_cus() ? 0 : 1;
        };
        int sq = size(square), up = size(update);
        // a round of 192 x 192 tiles is 9/4 of one of 128 x 128
        if (sq == 2 && 9 * cdiv(square[4], ns_cus()) <= 4 * cdiv(square[2], ns_cus())) sq = 4;
        auto place = [&](const int* at) { for (int i = 0; i < n; ++i) p.mat[i].tile0 = at[i]; };
        hipLaunchKernelGGL(ns_norm_kernel, dim3(NS_PARTS, n), dim3(256), 0, s, p);
        DVAE_LAUNCH_CHECK();
        place(split0);
        if (p.planes == 2) hipLaunchKernelGGL((ns_split_kernel<2>), dim3(split), dim3(256), 0, s, p);
        else hipLaunchKernelGGL((ns_split_kernel<1>), dim3(split), dim3(256), 0, s, p);
        DVAE_LAUNCH_CHECK();
#define NS_LAUNCH(TB, WN, KG, PL, NB, MODE, grid) \
    hipLaunchKernelGGL((ns_product_kernel<TB, WN, KG, PL, NB, MODE>), dim3(grid), dim3(128 * WN * KG), 0, s, group, 2 * (t & 1), t == 0)
#define NS_SMALL(PL, MODE, grid) hipLaunchKernelGGL((ns_small_kernel<PL, MODE>), dim3(grid), dim3(512), 0, s, group, 2 * (t & 1), t == 0)
#define NS_PRODUCT(set, MODE, size, grid)                                                 \
    do {                                                                                  \
        const NsGroup& group = set;                                                       \
        if (p.planes == 2) {                                                              \
            if (size == 3) NS_LAUNCH(256, 4, 1, 2, 2, MODE, grid);                        \
            else if (size == 4) NS_LAUNCH((MODE == NS_GRAM || MODE == NS_POLY ? 192 : 128), 2, 1, 2, (MODE == NS_GRAM || MODE == NS_POLY ? 3 : 2), MODE, grid); \
            else if (size == 2) NS_LAUNCH(128, 2, 1, 2, 2, MODE, grid);                   \
            else if (size == 0) NS_SMALL(2, MODE, grid);                                  \
            else if (grid <= ns_cus()) NS_LAUNCH(64, 2, 4, 2, 2, MODE, grid);             \
            else NS_LAUNCH(64, 2, 1, 2, 3, MODE, grid);                                   \
        } else {                                                                          \
            if (size == 3) NS_LAUNCH(256, 4, 1, 1, 2, MODE, grid);                        \
            else if (size == 4) NS_LAUNCH((MODE == NS_GRAM || MODE == NS_POLY ? 192 : 128), 2, 1, 1, (MODE == NS_GRAM || MODE == NS_POLY ? 3 : 2), MODE, grid); \
            else if (size == 2) NS_LAUNCH(128, 2, 1, 1, 2, MODE, grid);                   \
            else if (size == 0) NS_SMALL(1, MODE, grid);                                  \
            else if (grid <= ns_cus()) NS_LAUNCH(64, 2, 4, 1, 2, MODE, grid);             \
            else NS_LAUNCH(64, 2, 1, 1, 3, MODE, grid);                                   \
        }                                                                                 \
        DVAE_LAUNCH_CHECK();                                                              \
    } while (0)
        // X X^T of matrices with few rows in sets that take larger tiles: apart, on 64 x 64 tiles
        NsGroup most_of = p, few = p;
        int most_tiles = square[sq], few_tiles = 0;
        most_of.count = few.count = 0;
        if (p.planes == 2 && sq >= 2) {
            most_tiles = 0;
            for (int i = 0; i < n; ++i) {
                const bool is_few = p.mat[i].m() <= NS_FEW;
                NsGroup& group = is_few ? few : most_of;
                int& tiles = is_few ? few_tiles : most_tiles;
                group.mat[group.count] = p.mat[i];
                group.mat[group.count++].tile0 = tiles;
                const int mt = cdiv(ns_pad(p.mat[i].m(), p.pad), side[is_few ? 1 : sq]);
                tiles += mt * (mt + 1) / 2;
            }
        }
        for (int t = 0; t < steps; ++t) {
            p.a = coefficients[3 * t]; p.b = coefficients[3 * t + 1]; p.c = coefficients[3 * t + 2];
            p.shift = few.shift = most_of.shift = shift[t];
            place(square0[sq]);
            if (few_tiles == 0) NS_PRODUCT(p, NS_GRAM, sq, square[sq]);
            else {
                NS_PRODUCT(few, NS_GRAM, 1, few_tiles);
                if (most_tiles > 0) NS_PRODUCT(most_of, NS_GRAM, sq, most_tiles);
            }
            NS_PRODUCT(p, NS_POLY, sq, square[sq]);
            place(update0[up]);
            if (t + 1 < steps) NS_PRODUCT(p, NS_STEP, up, update[up]);
            else NS_PRODUCT(p, NS_LAST, up, update[up]);
        }
#undef NS_PRODUCT
#undef NS_LAUNCH
#undef NS_SMALL
    }
    return DVAE_OK;
}
