// Gated linear recurrence along packed sequences, with its backward pass, and its step for single tokens.
//
//   z_t = sigmoid(gate_t);   h_t = z_t h_{t-1} + (1 - z_t) x_t          per channel; h before a sequence: h0 or 0
//
// This is the state update of torch.nn.GRUCell (models.py:670: h' = (1 - z) n + z h) with a gate that does not look at the
// state, which makes the recurrence linear in h, and so a scan: a run of rows maps the state h before it to A h + B, with
// A = prod z, and two runs compose.  Backward, with e_t = dh_t (+ dlast at a sequence's last row):
//
//   G_t = e_t + z_{t+1} G_{t+1};   dx_t = (1 - z_t) G_t;   dgate_t = G_t (h_{t-1} - x_t) z_t (1 - z_t);   dh0 = z_first G_first
//
// the same kind of scan from the end.  h_{t-1} is not read back (it may have been rounded to 16 bits): the backward pass
// recomputes it in fp32 from the state before each tile, which the forward pass keeps.
//
// Layout: N rows (time, all sequences end to end) x D channels.  A workgroup's tile is W waves x RW rows by 64 V channels;
// each wave holds its RW rows in registers, the waves compose their (A, B) through LDS.  The tiles do not follow the
// sequences: a sequence's first row just makes A = 0, so that many short sequences and one long one cost the same.  All
// states, products and sums are fp32; outputs are rounded once.
#include "seq_common.h"

namespace dvae {

constexpr int TR = 64;  // rows of a tile: the state before every tile is kept for the backward pass

struct Rows {  // where the sequences lie
    const void* off;  // [S + 1] int32 / int64, or nullptr: S sequences of `len` rows each
    int i64;
    long S, len, N;
    __device__ __forceinline__ long at(long s) const {
        const long v = i64 ? reinterpret_cast<const int64_t*>(off)[s] : (long)reinterpret_cast<const int32_t*>(off)[s];
        return min(max(v, 0L), N);
    }
};

// What lane i (< RW) knows about row t0 + i, and the same as bit masks over the wave's rows.
struct Marks {
    unsigned start, end, cover;  // first / last row of its sequence; part of a sequence at all
    long seq;                    // this lane's row's sequence
};

template <int RW> __device__ __forceinline__ Marks mark_rows(const Rows& q, long t0) {
    const int lane = threadIdx.x & 63;
    const long t = t0 + lane;
    bool start = false, end = false, cover = false;
    long s = 0;
    if (lane < RW && t < q.N) {
        if (q.off) {
            long lo = 0, hi = q.S;  // the last s with off[s] <= t: empty sequences at the same row come before it
            while (lo < hi) {
                const long mid = (lo + hi + 1) >> 1;
                if (q.at(mid) <= t) lo = mid; else hi = mid - 1;
            }
            s = lo;
            if (s < q.S) {
                const long b = q.at(s), e = q.at(s + 1);
                cover = b <= t && t < e;
                start = cover && b == t;
                end = cover && e == t + 1;
            }
        } else {
            s = t / q.len;
            cover = true;
            start = t == s * q.len;
            end = t + 1 == (s + 1) * q.len;
        }
    }
    Marks m;
    m.start = (unsigned)__ballot(start);
    m.end = (unsigned)__ballot(end);
    m.cover = (unsigned)__ballot(cover);
    m.seq = s;
    return m;
}
__device__ __forceinline__ long seq_of(const Marks& m, int i) {
    const int lo = __builtin_amdgcn_readlane((int)m.seq, i), hi = __builtin_amdgcn_readlane((int)(m.seq >> 32), i);
    return ((long)hi << 32) | (unsigned)lo;
}

// z = sigmoid(g) and 1 - z.  The smaller of the two (at most 1/2) is exp(-|g|) / (1 + exp(-|g|)), good to a few ulp; the
// other is 1 minus it, good to half an ulp of 1 and unbiased, so that products of hundreds of z near 1 do not drift.
__device__ __forceinline__ void gate_of(float g, float& z, float& omz) {
    const float t = __expf(-fabsf(g));
    const float less = t * __builtin_amdgcn_rcpf(1.f + t), more = 1.f - less;
    z = g >= 0.f ? more : less;
    omz = g >= 0.f ? less : more;
}

// A run of rows as a map of the state (or of the gradient that flows back) before it: s -> A s + B.  A = 0 says that a
// sequence begins inside, so that nothing of s is left, not even a NaN; a product of gates is kept above 0 for that.
__device__ __forceinline__ float through(float A, float B, float s) { return A == 0.f ? B : fmaf(A, s, B); }
constexpr float A_MIN = 1.17549435e-38f;

// Carries between the tiles of a slab.  Every tile publishes its (A, B) per channel as soon as it has it, and then the
// state behind it as (0, state), which is the same map with everything before it folded in.  A tile looks back over up to
// LOOK published maps to the nearest whose A is 0 and applies the ones in between in order, oldest first: the sums are
// those of walking the tiles one by one, whatever the timing, so results do not vary.  64-bit relaxed atomics at device
// scope; a word that still holds the fill pattern has not been published, so no fences are needed.
constexpr int LOOK = 16;
constexpr unsigned long long UNSET = ~0ull;
__device__ __forceinline__ void publish(unsigned long long* at, float A, float B) {
    const unsigned long long w = ((unsigned long long)__float_as_uint(A) << 32) | __float_as_uint(B);
    __hip_atomic_store(at, w == UNSET ? w ^ 1 : w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// `ahead`: the words of the tiles before this one in walking order, nearest first, `step` apart; `count` of them exist.
__device__ __forceinline__ float look_back(const unsigned long long* nearest, long step, long count) {
    const int n = (int)min(count, (long)LOOK);
    for (int spin = 0; spin < (1 << 20); ++spin) {
        unsigned long long w[LOOK];
#pragma unroll
        for (int i = 0; i < LOOK; ++i)
            w[i] = i < n ? __hip_atomic_load(nearest + i * step, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
        int from = -1;  // the nearest whole state, if everything nearer is published
        bool open = true;
#pragma unroll
        for (int i = 0; i < LOOK; ++i) {
            if (w[i] == UNSET) open = false;
            // (past the first tile of all the state is zero)
            if (open && from < 0 && (i >= n ? count <= LOOK : (w[i] >> 32) == 0)) from = i;
        }
        if (open && from < 0 && count <= LOOK && n == LOOK) from = LOOK;
        if (__all(from >= 0)) {
            float s = 0.f;
#pragma unroll
            for (int i = LOOK - 1; i >= 0; --i)
                if (i <= from && i < n) s = through(__uint_as_float((unsigned)(w[i] >> 32)), __uint_as_float((unsigned)w[i]), s);
            return s;
        }
        __builtin_amdgcn_s_sleep(1);
    }
    return __uint_as_float(0x7FC00000u);  // not reached: every tile waits for earlier tickets only; NaN rather than a hang
}

struct ScanParams {
    const void *gate, *x, *dh;
    long ld_gate, ld_x, ld_dh;
    void *h, *dgate, *dx;           // contiguous [N][D]
    const float *h0, *dlast;        // [S][D] or nullptr
    float *last, *dh0;              // [S][D]
    float *states;                  // [tiles][D]: the state before each tile
    unsigned long long* words;      // [tiles][D]: a tile's map, as published
    unsigned* ticket;
    Rows q;
    int D, slabs;
};

template <int V> __device__ __forceinline__ void load_init(float (&h)[V], const float* p, long seq, int D, int c, bool live) {
#pragma unroll
    for (int j = 0; j < V; ++j) h[j] = p && live ? p[seq * D + c + j] : 0.f;
}

// Tiles are taken by ticket, in walking order: a tile's predecessors have always begun, so every wait ends.
__device__ __forceinline__ unsigned take_ticket(unsigned* ticket) {
    __shared__ unsigned mine;
    if (threadIdx.x == 0) mine = atomicAdd(ticket, 1u);
    __syncthreads();
    return mine;
}

template <typename T, int V, int RW, int W>
__global__ __launch_bounds__(W * 64) void scan_fwd_kernel(ScanParams p) {
    static_assert(RW * W == TR && W >= V, "");
    __shared__ float As[W][64 * V], Bs[W][64 * V], Cs[64 * V];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned unit = __builtin_amdgcn_readfirstlane(take_ticket(p.ticket));
    const int c0 = (int)(unit % (unsigned)p.slabs) * 64 * V, c = c0 + lane * V;
    const long tile = unit / (unsigned)p.slabs, t0 = tile * TR + wave * RW;
    const bool live = c < p.D;
    Pack<T, V> g[RW], x[RW];
#pragma unroll
    for (int i = 0; i < RW; ++i)
        if (live && t0 + i < p.q.N) {
            g[i] = load_pack<T, V>((const T*)p.gate + (t0 + i) * p.ld_gate + c);
            x[i] = load_pack<T, V>((const T*)p.x + (t0 + i) * p.ld_x + c);
        }
    const Marks m = mark_rows<RW>(p.q, t0);
    float A[V], h[V], z[RW][V], b[RW][V];
#pragma unroll
    for (int j = 0; j < V; ++j) { A[j] = 1.f; h[j] = 0.f; }
#pragma unroll
    for (int i = 0; i < RW; ++i) {
        if ((m.start >> i) & 1) {
            load_init<V>(h, p.h0, seq_of(m, i), p.D, c, live);
#pragma unroll
            for (int j = 0; j < V; ++j) A[j] = 0.f;
        }
        if ((m.cover >> i) & 1)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float omz;
                gate_of((float)g[i].e[j], z[i][j], omz);
                b[i][j] = omz * (float)x[i].e[j];
                h[j] = fmaf(z[i][j], h[j], b[i][j]);
                A[j] = A[j] == 0.f ? 0.f : fmaxf(A[j] * z[i][j], A_MIN);
            }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) { As[wave][lane * V + j] = A[j]; Bs[wave][lane * V + j] = h[j]; }
    __syncthreads();
    if (wave < V && c0 + (int)threadIdx.x < p.D) {  // one thread per channel from here to the barrier
        const int k = threadIdx.x;
        float a = 1.f, y = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            y = through(As[w][k], Bs[w][k], y);
            a = As[w][k] == 0.f ? 0.f : a == 0.f ? 0.f : fmaxf(a * As[w][k], A_MIN);
        }
        unsigned long long* word = p.words + tile * p.D + c0 + k;
        publish(word, a, y);
        const float s = tile == 0 ? 0.f : look_back(word - p.D, -(long)p.D, tile);
        if (a != 0.f) publish(word, 0.f, through(a, y, s));
        if (p.states) p.states[tile * p.D + c0 + k] = s;
        Cs[k] = s;
    }
    __syncthreads();
    if (!live) return;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        float s = Cs[lane * V + j];
        for (int w = 0; w < wave; ++w) s = through(As[w][lane * V + j], Bs[w][lane * V + j], s);
        h[j] = s;
    }
#pragma unroll
    for (int i = 0; i < RW; ++i) {
        if (t0 + i >= p.q.N) break;
        if ((m.start >> i) & 1) load_init<V>(h, p.h0, seq_of(m, i), p.D, c, live);
        const bool cover = (m.cover >> i) & 1;
        float o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (cover) h[j] = fmaf(z[i][j], h[j], b[i][j]);
            o[j] = cover ? h[j] : 0.f;
        }
        store_floats<T, V>((T*)p.h + (t0 + i) * p.D + c, o);
        if ((m.end >> i) & 1) {
            const long s = seq_of(m, i);
#pragma unroll
            for (int j = 0; j < V; ++j) p.last[s * p.D + c + j] = h[j];
        }
    }
}

// Backward: the tiles are walked from the last; what flows from a tile to the one before it is z_t G_t of its first row.
template <typename T, int V, int RW, int W>
__global__ __launch_bounds__(W * 64) void scan_bwd_kernel(ScanParams p) {
    static_assert(RW * W == TR && W >= V, "");
    __shared__ float As[W][64 * V], Bs[W][64 * V], Fs[W][64 * V], Cs[64 * V];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned unit = __builtin_amdgcn_readfirstlane(take_ticket(p.ticket));
    const int c0 = (int)(unit % (unsigned)p.slabs) * 64 * V, c = c0 + lane * V;
    const long tiles = (p.q.N + TR - 1) / TR, tile = tiles - 1 - unit / (unsigned)p.slabs, t0 = tile * TR + wave * RW;
    const bool live = c < p.D;
    Pack<T, V> g[RW], x[RW], d[RW];
#pragma unroll
    for (int i = 0; i < RW; ++i)
        if (live && t0 + i < p.q.N) {
            g[i] = load_pack<T, V>((const T*)p.gate + (t0 + i) * p.ld_gate + c);
            if (p.dh) d[i] = load_pack<T, V>((const T*)p.dh + (t0 + i) * p.ld_dh + c);
            x[i] = load_pack<T, V>((const T*)p.x + (t0 + i) * p.ld_x + c);
        }
    const Marks m = mark_rows<RW>(p.q, t0);
    auto row_grad = [&](int i, float (&e)[V]) {  // dh of row i, and dlast where the sequence ends
#pragma unroll
        for (int j = 0; j < V; ++j) e[j] = p.dh ? (float)d[i].e[j] : 0.f;
        if (((m.end >> i) & 1) && p.dlast) {
            const long s = seq_of(m, i);
#pragma unroll
            for (int j = 0; j < V; ++j) e[j] += live ? p.dlast[s * p.D + c + j] : 0.f;
        }
    };
    float A[V], B[V], h[V], z[RW][V], omz[RW][V];
#pragma unroll
    for (int j = 0; j < V; ++j) { A[j] = 1.f; B[j] = 0.f; h[j] = 0.f; }
#pragma unroll
    for (int i = 0; i < RW; ++i) {  // this wave's part of the forward scan
        if ((m.start >> i) & 1) load_init<V>(h, p.h0, seq_of(m, i), p.D, c, live);
        if ((m.cover >> i) & 1)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                gate_of((float)g[i].e[j], z[i][j], omz[i][j]);
                h[j] = fmaf(z[i][j], h[j], omz[i][j] * (float)x[i].e[j]);
            }
    }
#pragma unroll
    for (int i = RW - 1; i >= 0; --i)
        if ((m.cover >> i) & 1) {
            float e[V];
            row_grad(i, e);
            const bool first = (m.start >> i) & 1;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                B[j] = first ? 0.f : z[i][j] * (e[j] + B[j]);
                A[j] = first || A[j] == 0.f ? 0.f : fmaxf(A[j] * z[i][j], A_MIN);
            }
        }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        As[wave][lane * V + j] = A[j];
        Bs[wave][lane * V + j] = B[j];
        Fs[wave][lane * V + j] = h[j];
    }
    __syncthreads();
    if (wave < V && c0 + (int)threadIdx.x < p.D) {
        const int k = threadIdx.x;
        float a = 1.f, y = 0.f;
#pragma unroll
        for (int w = W - 1; w >= 0; --w) {
            y = through(As[w][k], Bs[w][k], y);
            a = As[w][k] == 0.f ? 0.f : a == 0.f ? 0.f : fmaxf(a * As[w][k], A_MIN);
        }
        unsigned long long* word = p.words + tile * p.D + c0 + k;
        publish(word, a, y);
        const float s = tile == tiles - 1 ? 0.f : look_back(word + p.D, p.D, tiles - 1 - tile);
        if (a != 0.f) publish(word, 0.f, through(a, y, s));
        Cs[k] = s;
    }
    __syncthreads();
    if (!live || t0 >= p.q.N) return;
    float C[V], prev[RW][V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        float s = p.states[tile * p.D + c + j];
        for (int w = 0; w < wave; ++w) s = through(As[w][lane * V + j], Fs[w][lane * V + j], s);
        h[j] = s;
        s = Cs[lane * V + j];
        for (int w = W - 1; w > wave; --w) s = through(As[w][lane * V + j], Bs[w][lane * V + j], s);
        C[j] = s;
    }
#pragma unroll
    for (int i = 0; i < RW; ++i) {
        if ((m.start >> i) & 1) load_init<V>(h, p.h0, seq_of(m, i), p.D, c, live);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            prev[i][j] = h[j];
            if ((m.cover >> i) & 1) h[j] = fmaf(z[i][j], h[j], omz[i][j] * (float)x[i].e[j]);
        }
    }
#pragma unroll
    for (int i = RW - 1; i >= 0; --i) {
        if (t0 + i >= p.q.N) continue;
        const bool cover = (m.cover >> i) & 1;
        float e[V], og[V], ox[V];
        row_grad(i, e);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float G = e[j] + C[j];
            og[j] = cover ? G * (prev[i][j] - (float)x[i].e[j]) * z[i][j] * omz[i][j] : 0.f;
            ox[j] = cover ? G * omz[i][j] : 0.f;
            if (cover) C[j] = z[i][j] * G;
        }
        store_floats<T, V>((T*)p.dgate + (t0 + i) * p.D + c, og);
        store_floats<T, V>((T*)p.dx + (t0 + i) * p.D + c, ox);
        if ((m.start >> i) & 1) {
            if (p.dh0) {
                const long s = seq_of(m, i);
#pragma unroll
                for (int j = 0; j < V; ++j) p.dh0[s * p.D + c + j] = C[j];
            }
#pragma unroll
            for (int j = 0; j < V; ++j) C[j] = 0.f;
        }
    }
}

// Before either pass: nothing is published yet, ticket 0 is next; and the sequences without rows, whose last state is the
// first (and whose gradient goes straight through).  Workgroups behind `fill_blocks` take four sequences each.
__global__ __launch_bounds__(256) void scan_begin_kernel(ulonglong2* __restrict__ words, long pairs, unsigned* __restrict__ ticket,
                                                         int fill_blocks, Rows q, const float* __restrict__ from,
                                                         float* __restrict__ to, int D) {
    if ((int)blockIdx.x < fill_blocks) {
        if (blockIdx.x == 0 && threadIdx.x == 0) *ticket = 0;
        for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < pairs; i += (long)fill_blocks * 256) words[i] = make_ulonglong2(UNSET, UNSET);
        return;
    }
    const long s = ((long)blockIdx.x - fill_blocks) * 4 + (threadIdx.x >> 6);
    if (s >= q.S || (q.off ? q.at(s) < q.at(s + 1) : q.len > 0)) return;
    for (int c = threadIdx.x & 63; c < D; c += 64) to[s * D + c] = from ? from[s * D + c] : 0.f;
}

// ------------------------------------------------------------------------------------------------------- single tokens
// One wave per row and slab.  Rows that name the same slot are advanced in their order by the first of them, so a
// repeated slot is neither a race nor dependent on timing; the search for them reads the slots alone.
template <typename T, int V>
__global__ __launch_bounds__(256) void scan_step_kernel(const T* __restrict__ gate, long ld_gate, const T* __restrict__ x, long ld_x,
                                                        float* __restrict__ state, long ld_state, long pool, const void* __restrict__ slots,
                                                        int i64, T* __restrict__ h, int B, int D, int slabs) {
    const int lane = threadIdx.x & 63;
    const long unit = (long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = (int)(unit / slabs), c = (int)(unit % slabs) * 64 * V + lane * V;
    if (b >= B) return;
    const bool live = c < D;
    auto slot = [&](int r) { return i64 ? reinterpret_cast<const int64_t*>(slots)[r] : (int64_t)reinterpret_cast<const int32_t*>(slots)[r]; };
    const long k = slots ? slot(b) : b;
    if (k < 0 || k >= pool) {  // padding
        const float zero[V] = {};
        if (live) store_floats<T, V>(h + (long)b * D + c, zero);
        return;
    }
    if (slots) {
        for (int r0 = 0; r0 < b; r0 += 64)
            if (__ballot(r0 + lane < b && slot(min(r0 + lane, b)) == k)) return;  // an earlier row advances this slot
    }
    float s[V];
    if (live)
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] = state[k * ld_state + c + j];
    auto advance = [&](int r) {
        if (!live) return;
        const Pack<T, V> g = load_pack<T, V>(gate + (long)r * ld_gate + c), y = load_pack<T, V>(x + (long)r * ld_x + c);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float z, omz;
            gate_of((float)g.e[j], z, omz);
            s[j] = fmaf(z, s[j], omz * (float)y.e[j]);
        }
        store_floats<T, V>(h + (long)r * D + c, s);
    };
    advance(b);
    if (slots)
        for (int r0 = b + 1; r0 < B; r0 += 64) {
            unsigned long long more = __ballot(r0 + lane < B && slot(min(r0 + lane, B - 1)) == k);
            while (more) {
                advance(r0 + __ffsll(more) - 1);
                more &= more - 1;
            }
        }
    if (live)
#pragma unroll
        for (int j = 0; j < V; ++j) state[k * ld_state + c + j] = s[j];
}

static int scan_check(const char* who, int64_t rows, int64_t seqs, const void* off, int32_t D, int32_t dtype) {
    DVAE_REQUIRE(known_dtype(dtype), "%s: unknown element type %d", who, dtype);
    DVAE_REQUIRE(rows >= 0 && rows < (1LL << 40), "%s: %lld rows are not supported", who, (long long)rows);
    DVAE_REQUIRE(seqs >= 0 && seqs < (1LL << 31), "%s: %lld sequences are not supported", who, (long long)seqs);
    DVAE_REQUIRE(D >= 1 && D <= (1 << 20), "%s: %d channels are not in 1 .. 2^20", who, D);
    DVAE_REQUIRE(off || (seqs > 0 ? rows % seqs == 0 : rows == 0), "%s: %lld rows are not %lld sequences of one length", who,
                 (long long)rows, (long long)seqs);
    return DVAE_OK;
}

struct ScanWs {
    int64_t words, bytes;  // [16 bytes: the ticket][words, to a whole number of 16 bytes]
    int64_t tiles;
};
static ScanWs scan_ws(int64_t rows, int64_t D) {
    ScanWs w;
    w.tiles = (rows + TR - 1) / TR;
    w.words = 16;
    w.bytes = w.words + (w.tiles * D + 1) / 2 * 16;
    return w;
}

// CALL(T, V, RW, W): V channels per lane, RW rows per wave (V * RW = 32 elements of every operand in registers), W waves
#define SCAN_BY_TYPE(dtype, vec, CALL)                                                          \
    do {                                                                                        \
        if ((dtype) == DVAE_F32) {                                                              \
            if ((vec) >= 2) { CALL(float, 2, 16, 4); } else { CALL(float, 1, 32, 2); }          \
        } else if ((dtype) == DVAE_BF16) {                                                      \
            if ((vec) >= 4) { CALL(__bf16, 4, 8, 8); }                                          \
            else if ((vec) == 2) { CALL(__bf16, 2, 16, 4); } else { CALL(__bf16, 1, 32, 2); }   \
        } else {                                                                                \
            if ((vec) >= 4) { CALL(_Float16, 4, 8, 8); }                                        \
            else if ((vec) == 2) { CALL(_Float16, 2, 16, 4); } else { CALL(_Float16, 1, 32, 2); } \
        }                                                                                       \
    } while (0)

static int scan_begin(ScanParams& p, void* ws, const ScanWs& L, const float* from, float* to, hipStream_t s) {
    p.ticket = (unsigned*)ws;
    p.words = (unsigned long long*)((char*)ws + L.words);
    const long pairs = (L.tiles * p.D + 1) / 2;
    const int fill = L.tiles == 0 ? 0 : (int)min((pairs + 255) / 256, 2048L);
    const bool empties = to && p.q.S > 0 && (p.q.off || p.q.len == 0);
    const long blocks = fill + (empties ? (p.q.S + 3) / 4 : 0);
    if (blocks == 0) return DVAE_OK;
    hipLaunchKernelGGL(scan_begin_kernel, dim3((unsigned)blocks), dim3(256), 0, s, (ulonglong2*)p.words, pairs, p.ticket, fill,
                       p.q, from, to, p.D);
    DVAE_LAUNCH_CHECK();
    return DVAE_OK;
}

}  // namespace dvae

extern "C" int64_t dvae_scan_state_floats(int64_t rows, int32_t D) {
    using namespace dvae;
    DVAE_TRY(scan_check("scan_state_floats", rows, 1, nullptr, D, DVAE_F32));
    return scan_ws(rows, D).tiles * D;
}
extern "C" int64_t dvae_scan_ws_bytes(int64_t rows, int32_t D) {
    using namespace dvae;
    DVAE_TRY(scan_check("scan_ws_bytes", rows, 1, nullptr, D, DVAE_F32));
    return scan_ws(rows, D).bytes;
}

extern "C" int dvae_scan_fwd(const void* gate, int64_t ld_gate, const void* x, int64_t ld_x, const void* off, int32_t off_i64,
                             const float* h0, void* h, float* last, float* states, void* ws, int64_t rows, int64_t seqs,
                             int32_t D, int32_t dtype, void* stream) {
    using namespace dvae;
    DVAE_TRY(scan_check("scan_fwd", rows, seqs, off, D, dtype));
    DVAE_REQUIRE((ld_gate == 0 || ld_gate >= D) && (ld_x == 0 || ld_x >= D), "scan_fwd: a row stride is below %d channels", D);
    DVAE_REQUIRE(rows == 0 || (gate && x && h && ws), "scan_fwd: null pointer");
    DVAE_REQUIRE(seqs == 0 || last, "scan_fwd: null pointer");
    DVAE_REQUIRE((uintptr_t)ws % 16 == 0, "scan_fwd: the workspace must be 16-byte aligned");
    hipStream_t s = (hipStream_t)stream;
    const ScanWs L = scan_ws(rows, D);
    const int vec = widest(elem_size(dtype), 8, {(int64_t)D, ld_gate, ld_x}, {gate, x, (const void*)h});
    ScanParams p = {};
    p.gate = gate; p.x = x; p.ld_gate = ld_gate; p.ld_x = ld_x; p.h = h; p.h0 = h0; p.last = last; p.states = states;
    p.q = {off, off_i64, seqs, seqs > 0 ? rows / seqs : 0, rows};
    p.D = D; p.slabs = cdiv(D, 64 * vec);
    DVAE_REQUIRE(L.tiles * p.slabs < (1LL << 31), "scan_fwd: %lld rows of %d channels are too many", (long long)rows, D);
    DVAE_TRY(scan_begin(p, ws, L, h0, last, s));
    if (rows == 0) return DVAE_OK;
    const dim3 grid((unsigned)(L.tiles * p.slabs));
#define SCAN_FWD(T, V, RW, W) hipLaunchKernelGGL((scan_fwd_kernel<T, V, RW, W>), grid, dim3(W * 64), 0, s, p)
    SCAN_BY_TYPE(dtype, vec, SCAN_FWD);
#undef SCAN_FWD
    DVAE_LAUNCH_CHECK();
    return DVAE_OK;
}

extern "C" int dvae_scan_bwd(const void* gate, int64_t ld_gate, const void* x, int64_t ld_x, const void* off, int32_t off_i64,
                             const float* h0, const float* states, const void* dh, int64_t ld_dh, const float* dlast, void* dgate,
                             void* dx, float* dh0, void* ws, int64_t rows, int64_t seqs, int32_t D, int32_t dtype, void* stream) {
    using namespace dvae;
    DVAE_TRY(scan_check("scan_bwd", rows, seqs, off, D, dtype));
    DVAE_REQUIRE((ld_gate == 0 || ld_gate >= D) && (ld_x == 0 || ld_x >= D) && (ld_dh == 0 || ld_dh >= D),
                 "scan_bwd: a row stride is below %d channels", D);
    DVAE_REQUIRE(rows == 0 || (gate && x && states && dgate && dx && ws), "scan_bwd: null pointer");
    DVAE_REQUIRE((uintptr_t)ws % 16 == 0, "scan_bwd: the workspace must be 16-byte aligned");
    hipStream_t s = (hipStream_t)stream;
    const ScanWs L = scan_ws(rows, D);
    const int vec = widest(elem_size(dtype), 8, {(int64_t)D, ld_gate, ld_x, dh ? ld_dh : 0},
                           {gate, x, dh, (const void*)dgate, (const void*)dx});
    ScanParams p = {};
    p.gate = gate; p.x = x; p.dh = dh; p.ld_gate = ld_gate; p.ld_x = ld_x; p.ld_dh = ld_dh;
    p.dgate = dgate; p.dx = dx; p.h0 = h0; p.dlast = dlast; p.dh0 = dh0; p.states = const_cast<float*>(states);
    p.q = {off, off_i64, seqs, seqs > 0 ? rows / seqs : 0, rows};
    p.D = D; p.slabs = cdiv(D, 64 * vec);
    DVAE_REQUIRE(L.tiles * p.slabs < (1LL << 31), "scan_bwd: %lld rows of %d channels are too many", (long long)rows, D);
    DVAE_TRY(scan_begin(p, ws, L, dlast, dh0, s));
    if (rows == 0) return DVAE_OK;
    const dim3 grid((unsigned)(L.tiles * p.slabs));
#define SCAN_BWD(T, V, RW, W) hipLaunchKernelGGL((scan_bwd_kernel<T, V, RW, W>), grid, dim3(W * 64), 0, s, p)
    SCAN_BY_TYPE(dtype, vec, SCAN_BWD);
#undef SCAN_BWD
    DVAE_LAUNCH_CHECK();
    return DVAE_OK;
}

extern "C" int dvae_scan_step(const void* gate, int64_t ld_gate, const void* x, int64_t ld_x, float* state, int64_t ld_state,
                              int64_t pool, const void* slots, int32_t slots_i64, void* h, int32_t rows, int32_t D, int32_t dtype,
                              void* stream) {
    using namespace dvae;
    DVAE_REQUIRE(known_dtype(dtype), "scan_step: unknown element type %d", dtype);
    DVAE_REQUIRE(rows >= 0 && rows <= (1 << 24) && pool >= 0, "scan_step: %d rows are not supported", rows);
    DVAE_REQUIRE(D >= 1 && D <= (1 << 20), "scan_step: %d channels are not in 1 .. 2^20", D);
    DVAE_REQUIRE((ld_gate == 0 || ld_gate >= D) && (ld_x == 0 || ld_x >= D) && ld_state >= D, "scan_step: a row stride is below %d channels", D);
    DVAE_REQUIRE(slots || rows <= pool, "scan_step: %d rows, but a pool of %lld states", rows, (long long)pool);
    if (rows == 0) return DVAE_OK;
    DVAE_REQUIRE(gate && x && h && (state || pool == 0), "scan_step: null pointer");
    const int vec = widest(elem_size(dtype), 8, {(int64_t)D, ld_gate, ld_x}, {gate, x, (const void*)h});
    const int slabs = cdiv(D, 64 * vec);
    const long units = (long)rows * slabs;
    DVAE_REQUIRE(units < (1LL << 31), "scan_step: %d rows of %d channels are too many", rows, D);
    const dim3 grid((unsigned)((units + 3) / 4));
#define SCAN_STEP(T, V, RW, W)                                                                                              \
    hipLaunchKernelGGL((scan_step_kernel<T, V>), grid, dim3(256), 0, (hipStream_t)stream, (const T*)gate, (long)ld_gate, (const T*)x, \
                       (long)ld_x, state, (long)ld_state, (long)pool, slots, slots_i64, (T*)h, rows, D, slabs)
    SCAN_BY_TYPE(dtype, vec, SCAN_STEP);
#undef SCAN_STEP
    DVAE_LAUNCH_CHECK();
    return DVAE_OK;
}
