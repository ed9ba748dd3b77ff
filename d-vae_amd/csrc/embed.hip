// Lookup of table rows by tokens, and the table's gradient from sorted tokens.
//
//   out[t]  = scale * W[id_t]                       (id outside [0, V): a row of zeros)
//   dW[v]   = scale * sum over t with id_t = v of dout[t]
//
// The one-hot vertex types of the GRU input (models.py:653, dvae_type_csr / dvae_type_colsum) are the same operation for
// at most 32 rows; here the table has any size.  Both directions are bound by HBM: the lookup reads N rows and writes N,
// the gradient reads N rows and writes V.
//
// Gradient, deterministic (no floating-point atomics):
//   1. the tokens are sorted by id, stably, so that equal tokens lie side by side in the order of their positions;
//   2. the sorted list is cut into chunks of EC tokens, one wave per chunk and column slab, whatever the tokens' counts (a
//      hot token is spread over as many waves as it fills chunks).  A run of equal tokens inside one chunk is summed in
//      registers and written once; a run that crosses a chunk's border leaves an fp32 partial per chunk;
//   3. the partials of each crossing run are added by the waves of one workgroup, each every so many of them in chunk order, and
//      the waves' sums in wave order: the same order every time.
// Rows that no token names are zeroed by further workgroups of launch 2, which find the tokens of their row range in the
// sorted list, so every row of dW is written exactly once.
//
// Measured at 65521 tokens of a 50001 x 1024 bf16 table (Zipf): lookup 39 us (6.0 TB/s of rows read and written, repeated
// rows from the caches), sorting 28 us in four launches, sums and zeros 60 us (236 MB, 3.9 TB/s), joining 12 us.  At 8192
// tokens of 8 rows of 501 floats: 7 us; 10, 7 and 5 us, far below the host's time for the calls.
#include "seq_common.h"

namespace dvae {

constexpr int EC = 32;              // sorted tokens per chunk (a multiple of ER, at most 62)
constexpr int ER = 8;               // rows in flight per wave
constexpr int SORT_ITEMS = 8;       // items per lane of a sorting tile
constexpr int SMALL_THREADS = 1024; // one workgroup sorts up to SMALL_THREADS * SORT_ITEMS tokens by itself
constexpr int SMALL_N = SMALL_THREADS * SORT_ITEMS;
constexpr int TILE_THREADS = 256;
constexpr int TILE_N = TILE_THREADS * SORT_ITEMS;
constexpr int MAX_SORT_BLOCKS = 256; // every block of a pass reads every block's digit counts
constexpr int ZERO_ROWS = 64;       // table rows per zeroing workgroup
constexpr int JOIN_THREADS = 512;

// ---------------------------------------------------------------------------------------------------------- lookup
__device__ __forceinline__ int token_key(const void* ids, int i64, long i, int V) {
    const long id = i64 ? reinterpret_cast<const int64_t*>(ids)[i] : (long)reinterpret_cast<const int32_t*>(ids)[i];
    return id >= 0 && id < V ? (int)id : V;
}

// one wave per row and pass; the lanes run along the row
template <typename T, int V>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const T* __restrict__ w, long ldw, const void* __restrict__ ids,
                                                        int i64, T* __restrict__ out, long n, int vocab, int D, float scale) {
    const int lane = threadIdx.x & 63;
    const long waves = (long)gridDim.x * (blockDim.x >> 6);
    for (long r = (long)blockIdx.x * (blockDim.x >> 6) + (threadIdx.x >> 6); r < n; r += waves) {
        const int k = __builtin_amdgcn_readfirstlane(token_key(ids, i64, r, vocab));
        const T* src = w + (long)k * ldw;
        T* dst = out + r * D;
        if (k < vocab) {
            for (int c = lane * V; c < D; c += 64 * V) {
                const Pack<T, V> v = load_pack<T, V>(src + c);
                float f[V];
#pragma unroll
                for (int i = 0; i < V; ++i) f[i] = (float)v.e[i] * scale;
                store_floats<T, V>(dst + c, f);
            }
        } else {
            const float f[V] = {};
            for (int c = lane * V; c < D; c += 64 * V) store_floats<T, V>(dst + c, f);
        }
    }
}

// --------------------------------------------------------------------------------------------------- sorting by token
// Radix sort, 8 bits a pass, least significant first; every pass is stable: equal tokens stay in the order of
// their positions, so that sums do not vary.  Bound by latency: up to SMALL_N tokens one workgroup does all passes, beyond that a pass is two launches.  Each wave takes 512 consecutive items in
// eight rounds of 64: the lanes with equal digits find each other by eight ballots, a lane's rank is the wave's count of
// its digit so far plus the number of such lanes below it.
__device__ __forceinline__ int wave_rank(unsigned digit, bool live, volatile int* cnt) {
    unsigned long long same = __ballot(live);
#pragma unroll
    for (int b = 0; b < 8; ++b) {
        const unsigned long long set = __ballot((digit >> b) & 1);
        same &= ((digit >> b) & 1) ? set : ~set;
    }
    const int lane = threadIdx.x & 63;
    const int below = __popcll(same & ((1ull << lane) - 1));
    int rank = 0;
    if (live) {
        const int before = cnt[digit];
        rank = before + below;
        if ((same >> lane) == 1ull) cnt[digit] = before + __popcll(same);  // the highest of them
    }
    __builtin_amdgcn_wave_barrier();
    return rank;
}

// exclusive sums of v over the 256 threads 0..255 of a workgroup; all threads call it
__device__ __forceinline__ int scan256(int v, int* wave_tot) {
    const int lane = threadIdx.x & 63;
    int x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o, 64);
        if (lane >= o) x += y;
    }
    if (lane == 63 && threadIdx.x < 256) wave_tot[threadIdx.x >> 6] = x;
    __syncthreads();
    if (threadIdx.x < 256)
        for (int w = 0; w < (int)(threadIdx.x >> 6); ++w) x += wave_tot[w];
    __syncthreads();
    return x - v;
}

// up to SMALL_N tokens: all passes in one workgroup, items in LDS between the passes
__global__ __launch_bounds__(SMALL_THREADS) void sort_small_kernel(const void* __restrict__ ids, int i64, int n, int V, int passes,
                                                                   int* __restrict__ key_out, int* __restrict__ pos_out) {
    constexpr int W = SMALL_THREADS / 64;
    __shared__ int lkey[SMALL_N], lpos[SMALL_N];
    __shared__ int cnt[W][256];
    __shared__ int wave_tot[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // the wave's share shrinks with n, so that small lists still use every wave
    const int rounds = (n + SMALL_THREADS - 1) / SMALL_THREADS;
    int key[SORT_ITEMS], pos[SORT_ITEMS], rank[SORT_ITEMS];
#pragma unroll
    for (int r = 0; r < SORT_ITEMS; ++r) {
        const int i = (wave * rounds + r) * 64 + lane;
        pos[r] = i;
        key[r] = r < rounds && i < n ? token_key(ids, i64, i, V) : 0;
    }
    for (int p = 0; p < passes; ++p) {
        for (int i = tid; i < W * 256; i += SMALL_THREADS) (&cnt[0][0])[i] = 0;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < SORT_ITEMS; ++r) {
            const int i = (wave * rounds + r) * 64 + lane;
            if (r < rounds) rank[r] = wave_rank((key[r] >> (8 * p)) & 255, i < n, cnt[wave]);
        }
        __syncthreads();
        int tot = 0;
        if (tid < 256)
            for (int w = 0; w < W; ++w) tot += cnt[w][tid];
        int run = scan256(tot, wave_tot);
        if (tid < 256)
            for (int w = 0; w < W; ++w) { const int t = cnt[w][tid]; cnt[w][tid] = run; run += t; }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < SORT_ITEMS; ++r) {
            const int i = (wave * rounds + r) * 64 + lane;
            if (r < rounds && i < n) {
                const int d = cnt[wave][(key[r] >> (8 * p)) & 255] + rank[r];
                lkey[d] = key[r];
                lpos[d] = pos[r];
            }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < SORT_ITEMS; ++r) {
            const int i = (wave * rounds + r) * 64 + lane;
            if (r < rounds && i < n) { key[r] = lkey[i]; pos[r] = lpos[i]; }
        }
        __syncthreads();
    }
#pragma unroll
    for (int r = 0; r < SORT_ITEMS; ++r) {
        const int i = (wave * rounds + r) * 64 + lane;
        if (r < rounds && i < n) { key_out[i] = key[r]; pos_out[i] = pos[r]; }
    }
}

// digit counts of pass p per block
__global__ __launch_bounds__(TILE_THREADS) void sort_count_kernel(const void* __restrict__ ids, int i64, const int* __restrict__ key_in,
                                                                  int n, int V, int p, int per_block, int* __restrict__ hist) {
    __shared__ int cnt[256];
    const int tid = threadIdx.x;
    cnt[tid] = 0;
    __syncthreads();
    const long beg = (long)blockIdx.x * per_block;
    const int end = (int)min((long)n, beg + per_block);
    for (long i = beg + tid; i < end; i += TILE_THREADS)
        atomicAdd(&cnt[((p == 0 ? token_key(ids, i64, i, V) : key_in[i]) >> (8 * p)) & 255], 1);
    __syncthreads();
    hist[(long)blockIdx.x * 256 + tid] = cnt[tid];
}

__global__ __launch_bounds__(TILE_THREADS) void sort_pass_kernel(const void* __restrict__ ids, int i64, const int* __restrict__ key_in,
                                                                 const int* __restrict__ pos_in, int n, int V, int p, int per_block,
                                                                 const int* __restrict__ hist, int* __restrict__ key_out,
                                                                 int* __restrict__ pos_out) {
    constexpr int W = TILE_THREADS / 64;
    __shared__ int cnt[W][256];
    __shared__ int wave_tot[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int before = 0, tot = 0;
    for (int b0 = 0; b0 < (int)gridDim.x; b0 += 16) {
        int h[16];
#pragma unroll
        for (int u = 0; u < 16; ++u) h[u] = hist[(long)min(b0 + u, (int)gridDim.x - 1) * 256 + tid];
#pragma unroll
        for (int u = 0; u < 16; ++u) {
            before += b0 + u < (int)blockIdx.x ? h[u] : 0;
            tot += b0 + u < (int)gridDim.x ? h[u] : 0;
        }
    }
    int base = scan256(tot, wave_tot) + before;  // where this block's items with digit `tid` begin
    const long beg = (long)blockIdx.x * per_block;
    const int end = (int)min((long)n, beg + per_block);
    for (long t0 = beg; t0 < end; t0 += TILE_N) {
#pragma unroll
        for (int w = 0; w < W; ++w) cnt[w][tid] = 0;
        __syncthreads();
        int key[SORT_ITEMS], pos[SORT_ITEMS], rank[SORT_ITEMS];
#pragma unroll
        for (int r = 0; r < SORT_ITEMS; ++r) {
            const long i = t0 + (wave * SORT_ITEMS + r) * 64 + lane;
            const bool live = i < end;
            key[r] = !live ? 0 : p == 0 ? token_key(ids, i64, i, V) : key_in[i];
            pos[r] = !live ? 0 : p == 0 ? (int)i : pos_in[i];
        }
#pragma unroll
        for (int r = 0; r < SORT_ITEMS; ++r)
            rank[r] = wave_rank((key[r] >> (8 * p)) & 255, t0 + (wave * SORT_ITEMS + r) * 64 + lane < end, cnt[wave]);
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) { const int t = cnt[w][tid]; cnt[w][tid] = base; base += t; }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < SORT_ITEMS; ++r)
            if (t0 + (wave * SORT_ITEMS + r) * 64 + lane < end) {
                const int d = cnt[wave][(key[r] >> (8 * p)) & 255] + rank[r];
                key_out[d] = key[r];
                pos_out[d] = pos[r];
            }
        __syncthreads();
    }
}

// first index of the sorted keys that is >= target; all 64 lanes probe, three steps for 262 144 keys
__device__ __forceinline__ int wave_lower_bound(const int* __restrict__ key, int n, int target) {
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = n;
    while (lo < hi) {
        const int step = (hi - lo + 63) / 64;
        const long i = lo + (long)(lane + 1) * step - 1;
        const int c = __popcll(__ballot(i < hi && key[i] < target));
        lo += c * step;
        if (step == 1) break;
        hi = min(hi, lo + step - 1);
    }
    return lo;
}

// ------------------------------------------------------------------------------------------------------ sums of rows
// Workgroups [0, sum_blocks): one wave per (chunk, slab of 64 V columns).  Workgroups behind them zero table rows.
template <typename T, int V>
__global__ __launch_bounds__(256) void embed_sum_kernel(const T* __restrict__ dout, long ldo, const int* __restrict__ key,
                                                        const int* __restrict__ pos, int n, int vocab, int D, float scale,
                                                        T* __restrict__ dw, float* __restrict__ part, int slabs, long units,
                                                        int sum_blocks) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if ((int)blockIdx.x >= sum_blocks) {
        __shared__ unsigned long long named;
        __shared__ int edge[2];
        const int r0 = ((int)blockIdx.x - sum_blocks) * ZERO_ROWS, rows = min(ZERO_ROWS, vocab - r0);
        if (threadIdx.x == 0) named = 0;
        if (wave < 2) {
            const int at = wave_lower_bound(key, n, wave == 0 ? r0 : r0 + rows);
            if (lane == 0) edge[wave] = at;
        }
        __syncthreads();
        int lo = edge[0], hi = edge[1];
        if (hi - lo <= 1024) {  // few tokens: all of them at once
            for (int i = lo + (int)threadIdx.x; i < hi; i += 256)
                if (i == lo || key[i] != key[i - 1]) atomicOr(&named, 1ull << (key[i] - r0));
        } else if (wave == 0) {  // a hot row among them: lane r looks for row r0 + r
            const int end = hi;
            while (lo < hi) {
                const int mid = lo + (hi - lo) / 2;
                if (key[mid] < r0 + lane) lo = mid + 1; else hi = mid;
            }
            const unsigned long long mask = __ballot(lo < end && key[min(lo, n - 1)] == r0 + lane);
            if (lane == 0) named = mask;
        }
        __syncthreads();
        const unsigned long long skip = named;
        const float f[V] = {};
        for (int r = wave; r < rows; r += 4)
            if (!((skip >> r) & 1))
                for (int c = lane * V; c < D; c += 64 * V) store_floats<T, V>(dw + (long)(r0 + r) * D + c, f);
        return;
    }
    const long unit = (long)blockIdx.x * 4 + wave;
    if (unit >= units) return;
    const int chunk = (int)(unit / slabs), c = (int)(unit % slabs) * 64 * V + lane * V;
    const int s = chunk * EC, e = min(n, s + EC);
    const bool live = c < D;
    const T* col = dout + (live ? c : D - V);  // idle lanes read the last columns
    // the chunk's tokens, one per lane; lanes 62 and 63 have the tokens on either side of it
    const int at = lane < EC ? min(s + lane, n - 1) : lane == 62 ? max(s - 1, 0) : min(e, n - 1);
    const int my_key = key[at], my_pos = pos[at];
    int cur = __builtin_amdgcn_readlane(my_key, 0);
    if (cur >= vocab) return;
    bool head = s > 0 && __builtin_amdgcn_readlane(my_key, 62) == cur;  // the run began in an earlier chunk
    float acc[V] = {};
    auto flush = [&](int which) {  // to the table's row, or to partial 0 (a run's continuation) or 1 (its begin)
        if (!live) return;
        if (which < 0) {
            float f[V];
#pragma unroll
            for (int j = 0; j < V; ++j) f[j] = acc[j] * scale;
            store_floats<T, V>(dw + (long)cur * D + c, f);
        } else {
            float* p = part + ((long)2 * chunk + which) * D + c;
#pragma unroll
            for (int j = 0; j < V; ++j) p[j] = acc[j];
        }
    };
    for (int i0 = s; i0 < e; i0 += ER) {
        Pack<T, V> row[ER];
        int k[ER];
#pragma unroll
        for (int u = 0; u < ER; ++u) {
            k[u] = i0 + u < e ? __builtin_amdgcn_readlane(my_key, i0 + u - s) : -1;
            row[u] = load_pack<T, V>(col + (long)__builtin_amdgcn_readlane(my_pos, i0 + u - s) * ldo);
        }
#pragma unroll
        for (int u = 0; u < ER; ++u) hold(row[u]);  // all ER rows are under way before the first is added
#pragma unroll
        for (int u = 0; u < ER; ++u) {
            if (k[u] != cur && k[u] >= 0) {
                flush(head ? 0 : -1);
                if (k[u] >= vocab) return;  // tokens outside the table sort last
                cur = k[u];
                head = false;
#pragma unroll
                for (int j = 0; j < V; ++j) acc[j] = 0.f;
            }
#pragma unroll
            for (int j = 0; j < V; ++j) acc[j] += k[u] >= 0 ? (float)row[u].e[j] : 0.f;
        }
    }
    flush(head ? 0 : e < n && __builtin_amdgcn_readlane(my_key, 63) == cur ? 1 : -1);
}

// The run that begins in this chunk and goes on in the next: its partials are summed per wave in chunk order, then the
// waves' sums in wave order.  The eight waves are G groups of 256 columns times 8 / G shares of the partials.
template <typename T>
__global__ __launch_bounds__(JOIN_THREADS) void embed_join_kernel(const int* __restrict__ key, int n, int vocab, int D, float scale,
                                                         T* __restrict__ dw, const float* __restrict__ part, int G) {
    constexpr int U = 8;
    __shared__ float sums[8][256];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int chunk = blockIdx.x, s = chunk * EC, e = s + EC;
    if (e >= n) return;
    const int k = key[e - 1];
    if (k >= vocab || key[e] != k || (s > 0 && key[s - 1] == k)) return;
    const int last = (wave_lower_bound(key, n, k + 1) - 1) / EC;
    const int shares = 8 / G, share = wave / G;
    for (int c0 = 0; c0 < D; c0 += G * 256) {
        const int c = c0 + (wave % G) * 256 + lane;
        float acc[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = share == 0 ? part[((long)2 * chunk + 1) * D + min(c + 64 * j, D - 1)] : 0.f;
        for (int q = chunk + 1 + share; q <= last; q += shares * U) {
            float v[U][4];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j) v[u][j] = part[(long)2 * min(q + u * shares, last) * D + min(c + 64 * j, D - 1)];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[j] += q + u * shares <= last ? v[u][j] : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; ++j) sums[wave][lane + 64 * j] = acc[j];
        __syncthreads();
        if (share == 0)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float t = acc[j];
                for (int w = wave + G; w < 8; w += G) t += sums[w][lane + 64 * j];
                if (c + 64 * j < D) dw[(long)k * D + c + 64 * j] = (T)(t * scale);
            }
    }
}

struct EmbedWs {
    int64_t key[2], pos[2], hist, part, bytes;  // byte offsets
    int passes, blocks, per_block, chunks;
};
static EmbedWs embed_ws(int64_t n, int64_t vocab, int64_t D) {
    EmbedWs w;
    w.passes = 1;
    while ((vocab >> (8 * w.passes)) != 0) ++w.passes;  // the keys run from 0 to vocab
    w.blocks = cdiv(n, TILE_N);
    if (w.blocks > MAX_SORT_BLOCKS) w.blocks = MAX_SORT_BLOCKS;
    w.per_block = n ? (int)(((n + w.blocks - 1) / w.blocks + TILE_N - 1) / TILE_N * TILE_N) : TILE_N;
    w.blocks = cdiv(n, w.per_block);
    w.chunks = cdiv(n, EC);
    const int64_t list = (n * 4 + 255) / 256 * 256;
    int64_t at = 0;
    for (int i = 0; i < 2; ++i) { w.key[i] = at; at += list; w.pos[i] = at; at += list; }
    w.hist = at;
    at += n > SMALL_N ? (int64_t)w.blocks * 1024 : 0;
    w.part = at;
    at += (int64_t)w.chunks * 2 * D * 4;
    w.bytes = at;
    return w;
}

static int embed_sizes(const char* who, int64_t n, int64_t vocab, int32_t D, int32_t dtype) {
    DVAE_REQUIRE(known_dtype(dtype), "%s: unknown element type %d", who, dtype);
    DVAE_REQUIRE(n >= 0 && n < (1LL << 31) - TILE_N * MAX_SORT_BLOCKS, "%s: %lld tokens are not supported", who, (long long)n);
    DVAE_REQUIRE(vocab >= 1 && vocab < (1LL << 31) - ZERO_ROWS, "%s: a table of %lld rows is not supported", who, (long long)vocab);
    DVAE_REQUIRE(D >= 1 && D <= (1 << 20), "%s: row length %d is not in 1 .. 2^20", who, D);
    return DVAE_OK;
}
// the gradient's launches: a workgroup per chunk of tokens, and one per ZERO_ROWS rows of the table
static int embed_grad_sizes(const char* who, int64_t n, int64_t vocab, int32_t D, int32_t dtype) {
    DVAE_TRY(embed_sizes(who, n, vocab, D, dtype));
    DVAE_REQUIRE(grid_fits((n + EC - 1) / EC, JOIN_THREADS), "%s: %lld tokens are not supported; at most 2^28 - 32", who, (long long)n);
    DVAE_REQUIRE(grid_fits((vocab + ZERO_ROWS - 1) / ZERO_ROWS, 256), "%s: a table of %lld rows is not supported; at most 2^30 - 64", who,
                 (long long)vocab);
    return DVAE_OK;
}

}  // namespace dvae

extern "C" int dvae_embed_fwd(const void* w, int64_t ld_w, const void* ids, int32_t ids_i64, void* out, int64_t n,
                              int64_t vocab, int32_t D, float scale, int32_t dtype, void* stream) {
    using namespace dvae;
    DVAE_TRY(embed_sizes("embed_fwd", n, vocab, D, dtype));
    DVAE_REQUIRE(ld_w >= D, "embed_fwd: row stride %lld is below the row length %d", (long long)ld_w, D);
    if (n == 0) return DVAE_OK;
    DVAE_REQUIRE(w && ids && out, "embed_fwd: null pointer");
    const int es = elem_size(dtype);
    const int vec = widest(es, 16, {(int64_t)D, ld_w}, {w, (const void*)out});
    const long blocks = (n + 3) / 4;
    const dim3 grid((unsigned)(blocks < 16384 ? blocks : 16384));
#define EMBED_FWD(T, V)                                                                                           \
    hipLaunchKernelGGL((embed_fwd_kernel<T, V>), grid, dim3(256), 0, (hipStream_t)stream, (const T*)w, (long)ld_w, \
                       ids, ids_i64, (T*)out, (long)n, (int)vocab, D, scale)
    DVAE_BY_TYPE(dtype, vec, EMBED_FWD);
#undef EMBED_FWD
    DVAE_LAUNCH_CHECK();
    return DVAE_OK;
}

extern "C" int64_t dvae_embed_bwd_ws_bytes(int64_t n, int64_t vocab, int32_t D) {
    using namespace dvae;
    DVAE_TRY(embed_grad_sizes("embed_bwd_ws_bytes", n, vocab, D, DVAE_F32));
    return embed_ws(n, vocab, D).bytes;
}

extern "C" int dvae_embed_bwd(const void* dout, int64_t ld_dout, const void* ids, int32_t ids_i64, void* dw, void* ws, int64_t n,
                              int64_t vocab, int32_t D, float scale, int32_t dtype, void* stream) {
    using namespace dvae;
    DVAE_TRY(embed_grad_sizes("embed_bwd", n, vocab, D, dtype));
    DVAE_REQUIRE(ld_dout == 0 || ld_dout >= D, "embed_bwd: row stride %lld is below the row length %d", (long long)ld_dout, D);
    DVAE_REQUIRE(dw, "embed_bwd: null pointer");
    DVAE_REQUIRE(n == 0 || (dout && ids && ws), "embed_bwd: null pointer");
    DVAE_REQUIRE((uintptr_t)ws % 16 == 0, "embed_bwd: the workspace must be 16-byte aligned");
    const EmbedWs L = embed_ws(n, vocab, D);
    const int es = elem_size(dtype);
    const int vec = widest(es, 16, {(int64_t)D, ld_dout}, {(const void*)dout, (const void*)dw});
    const int slabs = cdiv(D, 64 * vec), zero_blocks = cdiv(vocab, ZERO_ROWS);
    const long units = (long)L.chunks * slabs;
    const long sum_blocks = (units + 3) / 4;
    DVAE_REQUIRE(grid_fits(sum_blocks + zero_blocks, 256), "embed_bwd: %lld tokens of %d elements are too many", (long long)n, D);
    hipStream_t s = (hipStream_t)stream;
    char* b = (char*)ws;
    int at = 0;  // which of the two lists holds the sorted tokens
    if (n > 0 && n <= SMALL_N) {
        hipLaunchKernelGGL(sort_small_kernel, dim3(1), dim3(SMALL_THREADS), 0, s, ids, ids_i64, (int)n, (int)vocab, L.passes,
                           (int*)(b + L.key[0]), (int*)(b + L.pos[0]));
        DVAE_LAUNCH_CHECK();
    } else if (n > 0) {
        for (int p = 0; p < L.passes; ++p) {
            at = p & 1;
            const int *key_in = (const int*)(b + L.key[1 - at]), *pos_in = (const int*)(b + L.pos[1 - at]);
            hipLaunchKernelGGL(sort_count_kernel, dim3(L.blocks), dim3(TILE_THREADS), 0, s, ids, ids_i64, key_in, (int)n, (int)vocab, p,
                               L.per_block, (int*)(b + L.hist));
            DVAE_LAUNCH_CHECK();
            hipLaunchKernelGGL(sort_pass_kernel, dim3(L.blocks), dim3(TILE_THREADS), 0, s, ids, ids_i64, key_in, pos_in, (int)n,
                               (int)vocab, p, L.per_block, (const int*)(b + L.hist), (int*)(b + L.key[at]), (int*)(b + L.pos[at]));
            DVAE_LAUNCH_CHECK();
        }
    }
    const int* key = (const int*)(b + L.key[at]);
    const int* pos = (const int*)(b + L.pos[at]);
    float* part = (float*)(b + L.part);
#define EMBED_SUM(T, V)                                                                                                       \
    hipLaunchKernelGGL((embed_sum_kernel<T, V>), dim3((unsigned)(sum_blocks + zero_blocks)), dim3(256), 0, s, (const T*)dout, \
                       (long)ld_dout, key, pos, (int)n, (int)vocab, D, scale, (T*)dw, part, slabs, units, (int)sum_blocks)
    DVAE_BY_TYPE(dtype, vec, EMBED_SUM);
#undef EMBED_SUM
    DVAE_LAUNCH_CHECK();
    if (L.chunks > 1) {
        const int groups = D <= 256 ? 1 : D <= 512 ? 2 : D <= 1024 ? 4 : 8;
#define EMBED_JOIN(T)                                                                                                        \
    hipLaunchKernelGGL((embed_join_kernel<T>), dim3(L.chunks), dim3(JOIN_THREADS), 0, s, key, (int)n, (int)vocab, D, scale, (T*)dw, \
                       (const float*)part, groups)
        if (dtype == DVAE_F32) EMBED_JOIN(float);
        else if (dtype == DVAE_BF16) EMBED_JOIN(__bf16);
        else EMBED_JOIN(_Float16);
#undef EMBED_JOIN
        DVAE_LAUNCH_CHECK();
    }
    return DVAE_OK;
}
