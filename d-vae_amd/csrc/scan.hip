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
// sequences: a sequence's first row just makes A = -0, so that many short sequences and one long one cost the same.  All
// states, products and sums are fp32; outputs are rounded once.
//
// One pass over the data in either direction (forward 3, backward 5 matrices of memory traffic), tiles chained through
// look_back.  Measured on 131072 x 1024 bf16: forward 230 us (3.5 TB/s), backward 369 us (3.6 TB/s), where a large copy
// reaches 4.9.  With the look-back left out they take 187 and 272: what a tile waits for is two trips to device memory, its
// neighbours' maps and back, about 5 us of the 28 (17) that it lives, whatever the length of the chain: a second level of
// look-back over groups of 8 tiles, and other waves to publish than those that wait, made 223 and 354 of it, and 1 us more of a prompt.
// Forward tiles of 64 rows: 318 us (a longer chain), of 256: 239; backward of 128: 392 (fewer workgroups a CU).  A look-back of
// 16 tiles: 277 us forward (more words read per tile than it saves waits).
#include "seq_common.h"

namespace dvae {

constexpr int RW = 16;        // rows of a wave
constexpr int TRF = 128, TRB = 64;  // rows of a tile, forward and backward; the state before every TRB rows is kept for the latter

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

__device__ __forceinline__ Marks mark_rows(const Rows& q, long t0) {
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

// z = sigmoid(g) and 1 - z in one register: the smaller of the two (at most 1/2), negative where that is z.  It is
// exp(-|g|) / (1 + exp(-|g|)), good to a few ulp; the other is 1 minus it, good to half an ulp of 1 and unbiased, so that
// products of hundreds of z near 1 do not drift.
__device__ __forceinline__ float gate_code(float g) {
    const float t = __expf(-fabsf(g));
    const float less = t * __builtin_amdgcn_rcpf(1.f + t);
    return g >= 0.f ? less : -less;
}
__device__ __forceinline__ void gate_of_code(float code, float& z, float& omz) {
    const float less = fabsf(code), more = 1.f - less;
    const bool open = !(__float_as_uint(code) >> 31);
    z = open ? more : less;
    omz = open ? less : more;
}

// A run of rows as a map of the state (or of the gradient that flows back) before it: s -> A s + B.  A = -0 says that a
// sequence begins inside, so that nothing of s is left, not even a NaN; a product of gates is never below +0.  (Told from that by
// its sign, not by keeping products above 0: a state of 1e38, as inputs masked with their type's lowest value leave it, comes
// through the smallest number above 0 with a size of 1 behind gates that are closed.)
constexpr unsigned BEGINS = 0x80000000u;
__device__ __forceinline__ bool begins(float A) { return __float_as_uint(A) == BEGINS; }
__device__ __forceinline__ float through(float A, float B, float s) { return begins(A) ? B : fmaf(A, s, B); }
// two runs, the later one first
__device__ __forceinline__ float both(float A, float before) { return begins(A) || begins(before) ? __uint_as_float(BEGINS) : A * before; }

// Carries between the tiles of a slab.  Every tile publishes its (A, B) per channel as soon as it has it, and then the
// state behind it as (0, state), which is the same map with everything before it folded in.  A tile looks back over up to
// LOOK published maps to the nearest whose A is 0 and applies the ones in between in order, oldest first: the sums are
// those of walking the tiles one by one, whatever the timing, so results do not vary.  64-bit relaxed atomics at device
// scope; a word that still holds the fill pattern has not been published, so no fences are needed.
constexpr int LOOK = 8;
constexpr unsigned long long UNSET = ~0ull;
constexpr long FILL_BLOCKS = 2048;  // at most, before a pass
constexpr int SPINS = 1 << 22;  // never reached: every tile waits for earlier tickets only; else the states from there on are NaN, not a hang
__device__ __forceinline__ void publish(unsigned long long* at, float A, float B) {
    const unsigned long long w = ((unsigned long long)__float_as_uint(A) << 32) | __float_as_uint(B);
    __hip_atomic_store(at, w == UNSET ? w ^ 1 : w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ unsigned long long read_word(const unsigned long long* at) {
    return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// The state that flows into a tile.  `nearest`: the word of the tile before it in walking order, the others `step` apart,
// `count` of them.  All words in reach are read at once; where none is whole yet, the farthest one is the next to become
// so, and only that one is polled.
__device__ __forceinline__ float look_back(const unsigned long long* nearest, long step, long count) {
    const int n = (int)min(count, (long)LOOK);
    unsigned long long w[LOOK];
    int spins = 0;
    bool open;
    do {
        open = true;
#pragma unroll
        for (int i = 0; i < LOOK; ++i) w[i] = i < n ? read_word(nearest + i * step) : (unsigned long long)BEGINS << 32;
#pragma unroll
        for (int i = 0; i < LOOK; ++i) {
            open = open && w[i] != UNSET;
            if ((w[i] >> 32) == BEGINS) break;  // whole: nothing farther matters
        }
    } while (!__all(open) && ++spins < SPINS);
    bool whole = count < LOOK;
#pragma unroll
    for (int i = 0; i < LOOK; ++i) whole = whole || (w[i] >> 32) == BEGINS;
    if (count == LOOK) whole = true;
    while (!__all(whole) && ++spins < SPINS) {
        __builtin_amdgcn_s_sleep(1);
        const unsigned long long far = read_word(nearest + (LOOK - 1) * step);
        if (!whole && (far >> 32) == BEGINS) { w[LOOK - 1] = far; whole = true; }
    }
    float s = spins < SPINS ? 0.f : __uint_as_float(0x7FC00000u);
#pragma unroll
    for (int i = LOOK - 1; i >= 0; --i)
        if (i < n) s = through(__uint_as_float((unsigned)(w[i] >> 32)), __uint_as_float((unsigned)w[i]), s);
    return s;
}

struct ScanParams {
    const void *gate, *x, *dh;
    long ld_gate, ld_x, ld_dh;
    void *h, *dgate, *dx;           // contiguous [N][D]
    const float *h0, *dlast;        // [S][D] or nullptr
    float *last, *dh0;              // [S][D]
    float *states;                  // [N / TRB rounded up][D]: the state before every TRB rows
    unsigned long long* words;      // [tiles][D]: a tile's map, as published
    unsigned* ticket;               // nullptr: one tile
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

// A wave's rows of one matrix: a buffer based at its first row, the lane's columns as the one vector offset, the row as a
// scalar offset, so that no lane computes an address.  Rows beyond the last and columns beyond D are read from the nearest
// inside and not used: loads without branches.
template <typename T, int V> struct RowBuffer {
    __amdgpu_buffer_rsrc_t rsrc;
    unsigned col, pitch;  // bytes
    int most;             // rows behind the first that may be touched
    __device__ __forceinline__ RowBuffer(const void* base, long ld, long t0, long N, int c) {
        const long first = min(t0, N - 1);
        rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)((const T*)base + first * ld), 0, 0x7FFFFFFF, 0x00020000);
        col = (unsigned)c * sizeof(T);
        pitch = (unsigned)(ld * sizeof(T));
        most = (int)min(N - 1 - first, 63L);
    }
    __device__ __forceinline__ Pack<T, V> load(int i) const {
        const unsigned at = min(i, most) * pitch;
        if constexpr (sizeof(T) * V == 4) return __builtin_bit_cast(Pack<T, V>, __builtin_amdgcn_raw_buffer_load_b32(rsrc, col, at, 0));
        else return __builtin_bit_cast(Pack<T, V>, __builtin_amdgcn_raw_buffer_load_b16(rsrc, col, at, 0));
    }
    __device__ __forceinline__ void store(int i, const float (&f)[V]) const {
        Pack<T, V> o;
#pragma unroll
        for (int j = 0; j < V; ++j) o.e[j] = (T)f[j];
        if constexpr (sizeof(T) * V == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, o), rsrc, col, i * pitch, 0);
        else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, o), rsrc, col, i * pitch, 0);
    }
};
template <typename T, int V>
__device__ __forceinline__ void load_rows(Pack<T, V> (&r)[RW], const void* base, long ld, long t0, long N, int D, int c) {
    const RowBuffer<T, V> b(base, ld, t0, N, min(c, D - V));
#pragma unroll
    for (int i = 0; i < RW; ++i) r[i] = b.load(i);
}

// The sequences without rows: the state behind them is the one before (and their gradient goes straight through).
// Workgroup `block` takes four sequences.
__device__ __forceinline__ void pass_empty(const Rows& q, long block, const float* from, float* to, int D) {
    for (int u = 0; u < 4; ++u) {
        const long s = block * 4 + u;
        if (s >= q.S || (q.off ? q.at(s) < q.at(s + 1) : q.len > 0)) continue;
        for (int c = threadIdx.x; c < D; c += blockDim.x) to[s * D + c] = from ? from[s * D + c] : 0.f;
    }
}

struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };

// Where a wave's rows all lie inside one sequence (PLAIN below) the row loops have no branches, so that the loads, the
// exponentials and the chains of multiply-adds of several channels overlap.
template <typename T, int V>
__global__ __launch_bounds__(TRF / RW * 64) void scan_fwd_kernel(ScanParams p) {
    constexpr int W = TRF / RW;
    static_assert(W >= V, "");
    __shared__ float As[W][64 * V], Bs[W][64 * V], Cs[64 * V];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (!p.ticket && (int)blockIdx.x >= p.slabs) return pass_empty(p.q, (long)blockIdx.x - p.slabs, p.h0, p.last, p.D);
    const unsigned unit = p.ticket ? __builtin_amdgcn_readfirstlane(take_ticket(p.ticket)) : blockIdx.x;
    const int c0 = (int)(unit % (unsigned)p.slabs) * 64 * V, c = c0 + lane * V;
    const long tile = unit / (unsigned)p.slabs, t0 = tile * TRF + wave * RW;
    const bool live = c < p.D;
    Pack<T, V> g[RW], x[RW];
    load_rows<T, V>(g, p.gate, p.ld_gate, t0, p.q.N, p.D, c);
    load_rows<T, V>(x, p.x, p.ld_x, t0, p.q.N, p.D, c);
    const Marks m = mark_rows(p.q, t0);
    const bool plain = m.start == 0 && m.end == 0 && m.cover == (unsigned)((1ull << RW) - 1);
    float A[V], h[V], code[RW][V];
#pragma unroll
    for (int j = 0; j < V; ++j) { A[j] = 1.f; h[j] = 0.f; }
#pragma unroll
    for (int i = 0; i < RW; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) code[i][j] = gate_code((float)g[i].e[j]);
    auto local = [&](auto mixed) {
#pragma unroll
        for (int i = 0; i < RW; ++i) {
            if (decltype(mixed)::value) {
                if ((m.start >> i) & 1) load_init<V>(h, p.h0, seq_of(m, i), p.D, c, live);
                if (!((m.cover >> i) & 1)) continue;
            }
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float z, omz;
                gate_of_code(code[i][j], z, omz);
                h[j] = fmaf(z, h[j], omz * (float)x[i].e[j]);
                A[j] *= z;
            }
        }
    };
    if (plain) local(No()); else local(Yes());
#pragma unroll
    for (int j = 0; j < V; ++j) {
        As[wave][lane * V + j] = m.start ? __uint_as_float(BEGINS) : A[j];
        Bs[wave][lane * V + j] = h[j];
    }
    __syncthreads();
    if (wave < V && c0 + (int)threadIdx.x < p.D) {  // one thread per channel from here to the barrier
        const int k = threadIdx.x;
        float a = 1.f, y = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            y = through(As[w][k], Bs[w][k], y);
            a = both(As[w][k], a);
        }
        unsigned long long* word = p.words + tile * p.D + c0 + k;
        publish(word, a, y);
        const float s = tile == 0 ? 0.f : look_back(word - p.D, -(long)p.D, tile);
        if (!begins(a)) publish(word, __uint_as_float(BEGINS), through(a, y, s));
        Cs[k] = s;
    }
    __syncthreads();
    if (!live) return;
#pragma unroll
    for (int i = 0; i < RW; ++i) {
        hold(x[i]);
#pragma unroll
        for (int j = 0; j < V; ++j) hold(code[i][j]);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        float s = Cs[lane * V + j];
        for (int w = 0; w < wave; ++w) s = through(As[w][lane * V + j], Bs[w][lane * V + j], s);
        h[j] = s;
    }
    if (p.states && wave % (TRB / RW) == 0 && t0 < p.q.N)
#pragma unroll
        for (int j = 0; j < V; ++j) p.states[t0 / TRB * p.D + c + j] = h[j];
    const RowBuffer<T, V> out(p.h, p.D, t0, p.q.N, c);
    auto apply = [&](auto mixed) {
#pragma unroll
        for (int i = 0; i < RW; ++i) {
            bool cover = true;
            if (decltype(mixed)::value) {
                if (t0 + i >= p.q.N) continue;
                if ((m.start >> i) & 1) load_init<V>(h, p.h0, seq_of(m, i), p.D, c, live);
                cover = (m.cover >> i) & 1;
            }
            float o[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float z, omz;
                gate_of_code(code[i][j], z, omz);
                if (cover) h[j] = fmaf(z, h[j], omz * (float)x[i].e[j]);
                o[j] = cover ? h[j] : 0.f;
            }
            out.store(i, o);
            if (decltype(mixed)::value && ((m.end >> i) & 1)) {
                const long s = seq_of(m, i);
#pragma unroll
                for (int j = 0; j < V; ++j) p.last[s * p.D + c + j] = h[j];
            }
        }
    };
    if (plain) apply(No()); else apply(Yes());
}

// Backward: the tiles are walked from the last; what flows from a tile to the one before it is z_t G_t of its first row.
template <typename T, int V>
__global__ __launch_bounds__(TRB / RW * 64) void scan_bwd_kernel(ScanParams p) {
    constexpr int W = TRB / RW;
    static_assert(W >= V, "");
    __shared__ float As[W][64 * V], Bs[W][64 * V], Fs[W][64 * V], Cs[64 * V];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (!p.ticket && (int)blockIdx.x >= p.slabs) return pass_empty(p.q, (long)blockIdx.x - p.slabs, p.dlast, p.dh0, p.D);
    const unsigned unit = p.ticket ? __builtin_amdgcn_readfirstlane(take_ticket(p.ticket)) : blockIdx.x;
    const int c0 = (int)(unit % (unsigned)p.slabs) * 64 * V, c = c0 + lane * V;
    const long tiles = (p.q.N + TRB - 1) / TRB, tile = tiles - 1 - unit / (unsigned)p.slabs, t0 = tile * TRB + wave * RW;
    const bool live = c < p.D;
    Pack<T, V> g[RW], x[RW], d[RW];
    load_rows<T, V>(g, p.gate, p.ld_gate, t0, p.q.N, p.D, c);
    load_rows<T, V>(x, p.x, p.ld_x, t0, p.q.N, p.D, c);
    if (p.dh) load_rows<T, V>(d, p.dh, p.ld_dh, t0, p.q.N, p.D, c);
    else
#pragma unroll
        for (int i = 0; i < RW; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) d[i].e[j] = (T)0.f;
    float begin[V];  // the state before the tile
#pragma unroll
    for (int j = 0; j < V; ++j) begin[j] = p.states[tile * p.D + min(c, p.D - V) + j];
    const Marks m = mark_rows(p.q, t0);
    const bool plain = m.start == 0 && m.end == 0 && m.cover == (unsigned)((1ull << RW) - 1);
    auto row_grad = [&](auto mixed, int i, float (&e)[V]) {  // dh of row i, and dlast where the sequence ends
#pragma unroll
        for (int j = 0; j < V; ++j) e[j] = (float)d[i].e[j];
        if (decltype(mixed)::value && ((m.end >> i) & 1) && p.dlast) {
            const long s = seq_of(m, i);
#pragma unroll
            for (int j = 0; j < V; ++j) e[j] += live ? p.dlast[s * p.D + c + j] : 0.f;
        }
    };
    float A[V], B[V], h[V], code[RW][V];
#pragma unroll
    for (int j = 0; j < V; ++j) { A[j] = 1.f; B[j] = 0.f; h[j] = 0.f; }
#pragma unroll
    for (int i = 0; i < RW; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) code[i][j] = gate_code((float)g[i].e[j]);
    auto local = [&](auto mixed) {
#pragma unroll
        for (int i = 0; i < RW; ++i) {  // this wave's part of the forward scan
            if (decltype(mixed)::value) {
                if ((m.start >> i) & 1) load_init<V>(h, p.h0, seq_of(m, i), p.D, c, live);
                if (!((m.cover >> i) & 1)) continue;
            }
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float z, omz;
                gate_of_code(code[i][j], z, omz);
                h[j] = fmaf(z, h[j], omz * (float)x[i].e[j]);
            }
        }
#pragma unroll
        for (int i = RW - 1; i >= 0; --i) {
            if (decltype(mixed)::value && !((m.cover >> i) & 1)) continue;
            float e[V];
            row_grad(mixed, i, e);
            const bool first = decltype(mixed)::value && ((m.start >> i) & 1);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float z, omz;
                gate_of_code(code[i][j], z, omz);
                B[j] = first ? 0.f : z * (e[j] + B[j]);
                A[j] *= z;
            }
        }
    };
    if (plain) local(No()); else local(Yes());
#pragma unroll
    for (int j = 0; j < V; ++j) {
        As[wave][lane * V + j] = m.start ? __uint_as_float(BEGINS) : A[j];
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
            a = both(As[w][k], a);
        }
        unsigned long long* word = p.words + tile * p.D + c0 + k;
        publish(word, a, y);
        const float s = tile == tiles - 1 ? 0.f : look_back(word + p.D, p.D, tiles - 1 - tile);
        if (!begins(a)) publish(word, __uint_as_float(BEGINS), through(a, y, s));
        Cs[k] = s;
    }
    __syncthreads();
    if (!live || t0 >= p.q.N) return;
#pragma unroll
    for (int i = 0; i < RW; ++i) {
        hold(x[i]);
        hold(d[i]);
#pragma unroll
        for (int j = 0; j < V; ++j) hold(code[i][j]);
    }
    float C[V], prev[RW][V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        float s = begin[j];
        for (int w = 0; w < wave; ++w) s = through(As[w][lane * V + j], Fs[w][lane * V + j], s);
        h[j] = s;
        s = Cs[lane * V + j];
        for (int w = W - 1; w > wave; --w) s = through(As[w][lane * V + j], Bs[w][lane * V + j], s);
        C[j] = s;
    }
    const RowBuffer<T, V> out_gate(p.dgate, p.D, t0, p.q.N, c), out_x(p.dx, p.D, t0, p.q.N, c);
    auto apply = [&](auto mixed) {
#pragma unroll
        for (int i = 0; i < RW; ++i) {
            if (decltype(mixed)::value && ((m.start >> i) & 1)) load_init<V>(h, p.h0, seq_of(m, i), p.D, c, live);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                prev[i][j] = h[j];
                float z, omz;
                gate_of_code(code[i][j], z, omz);
                if (!decltype(mixed)::value || ((m.cover >> i) & 1)) h[j] = fmaf(z, h[j], omz * (float)x[i].e[j]);
            }
        }
#pragma unroll
        for (int i = RW - 1; i >= 0; --i) {
            if (decltype(mixed)::value && t0 + i >= p.q.N) continue;
            const bool cover = !decltype(mixed)::value || ((m.cover >> i) & 1);
            float e[V], og[V], ox[V];
            row_grad(mixed, i, e);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float z, omz;
                gate_of_code(code[i][j], z, omz);
                const float G = e[j] + C[j];
                // (the gates first: z (1 - z) keeps what a closed one meets, an input of its type's lowest value, from overflowing)
                og[j] = cover ? G * z * omz * (prev[i][j] - (float)x[i].e[j]) : 0.f;
                ox[j] = cover ? G * omz : 0.f;
                if (cover) C[j] = z * G;
            }
            out_gate.store(i, og);
            out_x.store(i, ox);
            if (decltype(mixed)::value && ((m.start >> i) & 1)) {
                if (p.dh0) {
                    const long s = seq_of(m, i);
#pragma unroll
                    for (int j = 0; j < V; ++j) p.dh0[s * p.D + c + j] = C[j];
                }
#pragma unroll
                for (int j = 0; j < V; ++j) C[j] = 0.f;
            }
        }
    };
    if (plain) apply(No()); else apply(Yes());
}

// Before a pass over several tiles: nothing is published yet, ticket 0 is next; and the sequences without rows, by the
// workgroups behind `fill_blocks`.  A single tile per slab has nothing to wait for: no tickets, no look-back, and the
// sequences without rows are taken by workgroups behind the tiles' (100 rows of 501 floats: 9.2 -> 6.9 us).
__global__ __launch_bounds__(256) void scan_begin_kernel(ulonglong2* __restrict__ words, long pairs, unsigned* __restrict__ ticket,
                                                         int fill_blocks, Rows q, const float* __restrict__ from,
                                                         float* __restrict__ to, int D) {
    if ((int)blockIdx.x < fill_blocks) {
        if (blockIdx.x == 0 && threadIdx.x == 0) *ticket = 0;
        for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < pairs; i += (long)fill_blocks * 256) words[i] = make_ulonglong2(UNSET, UNSET);
        return;
    }
    pass_empty(q, (long)blockIdx.x - fill_blocks, from, to, D);
}

// ------------------------------------------------------------------------------------------------------- single tokens
// Bound by memory for large batches (2048 rows of 1024 bf16: 9.3 us; without slots 6.1 us, 4.8 TB/s), by the launch for small.
// One wave per row and slab.  Rows that name the same slot are advanced in their order by the first of them, so a
// repeated slot is neither a race nor dependent on timing; the search for them reads the slots alone.
template <typename I> struct Slots4 { I s[4]; };  // (aligned to one slot only)

template <typename T, int V, typename I>
__global__ __launch_bounds__(256) void scan_step_kernel(const T* __restrict__ gate, long ld_gate, const T* __restrict__ x, long ld_x,
                                                        float* __restrict__ state, long ld_state, long pool, const I* __restrict__ slots,
                                                        T* __restrict__ h, int B, int D, int slabs) {
    const int lane = threadIdx.x & 63;
    const long unit = (long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = (int)(unit / slabs), c = (int)(unit % slabs) * 64 * V + lane * V;
    if (b >= B) return;
    const bool live = c < D;
    const long k = slots ? (long)slots[b] : b;
    if (k < 0 || k >= pool) {  // padding
        const float zero[V] = {};
        if (live) store_floats<T, V>(h + (long)b * D + c, zero);
        return;
    }
    // the row and the state are under way while the slots are searched; a row that is not the first of its slot drops them
    const int cc = live ? c : D - V;
    Pack<T, V> g = load_pack<T, V>(gate + (long)b * ld_gate + cc), y = load_pack<T, V>(x + (long)b * ld_x + cc);
    float s[V];
#pragma unroll
    for (int j = 0; j < V; ++j) s[j] = state[k * ld_state + cc + j];
    bool again = false;  // a later row names the same slot
    if (slots) {
        const I mine = (I)k;
        bool before = false, after = false;
        // four slots a lane and load, four loads under way; the last loads end at B, rows seen twice do no harm
        for (int r0 = 0; B >= 256 && r0 < B; r0 += 1024) {
            Slots4<I> q[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) q[u] = *reinterpret_cast<const Slots4<I>*>(slots + min(r0 + 256 * u, B - 256) + lane * 4);
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = min(r0 + 256 * u, B - 256) + lane * 4 + e;
                    before = before || (q[u].s[e] == mine && r < b);
                    after = after || (q[u].s[e] == mine && r > b);
                }
        }
        if (B < 256)
            for (int r0 = 0; r0 < B; r0 += 64) {
                const int r = r0 + lane;
                const bool same = r < B && slots[min(r, B - 1)] == mine;
                before = before || (same && r < b);
                after = after || (same && r > b);
            }
        if (__any(before)) return;  // an earlier row advances this slot
        again = __any(after);
    }
    auto advance = [&](int r) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float z, omz;
            gate_of_code(gate_code((float)g.e[j]), z, omz);
            s[j] = fmaf(z, s[j], omz * (float)y.e[j]);
        }
        if (live) store_floats<T, V>(h + (long)r * D + c, s);
    };
    advance(b);
    if (again)
        for (int r0 = b + 1; r0 < B; r0 += 64) {
            unsigned long long more = __ballot(r0 + lane < B && (long)slots[min(r0 + lane, B - 1)] == k);
            while (more) {
                const int r = r0 + __ffsll(more) - 1;
                g = load_pack<T, V>(gate + (long)r * ld_gate + cc);
                y = load_pack<T, V>(x + (long)r * ld_x + cc);
                advance(r);
                more &= more - 1;
            }
        }
    if (live)
#pragma unroll
        for (int j = 0; j < V; ++j) state[k * ld_state + c + j] = s[j];
}

static int scan_check(const char* who, int64_t rows, int64_t seqs, const void* off, int64_t ld_most, int32_t D, int32_t dtype) {
    DVAE_REQUIRE(known_dtype(dtype), "%s: unknown element type %d", who, dtype);
    DVAE_REQUIRE(rows >= 0 && rows < (1LL << 40), "%s: %lld rows are not supported", who, (long long)rows);
    DVAE_REQUIRE(seqs >= 0 && seqs < (1LL << 31), "%s: %lld sequences are not supported", who, (long long)seqs);
    DVAE_REQUIRE(D >= 1 && D <= (1 << 20), "%s: %d channels are not in 1 .. 2^20", who, D);
    // (a wave addresses its 16 rows with 32-bit byte offsets)
    DVAE_REQUIRE(ld_most <= (1 << 23), "%s: a row stride of %lld elements is not supported", who, (long long)ld_most);
    DVAE_REQUIRE(off || (seqs > 0 ? rows % seqs == 0 : rows == 0), "%s: %lld rows are not %lld sequences of one length", who,
                 (long long)rows, (long long)seqs);
    return DVAE_OK;
}

struct ScanWs {
    int64_t words, bytes;  // [16 bytes: the ticket][words, to a whole number of 16 bytes]; enough for either direction
    int64_t tiles, states;
};
static ScanWs scan_ws(int64_t rows, int64_t D, int tile_rows) {
    ScanWs w;
    w.tiles = (rows + tile_rows - 1) / tile_rows;
    w.states = (rows + TRB - 1) / TRB * D;
    w.words = 16;
    w.bytes = w.words + (w.states + 1) / 2 * 16;
    return w;
}

// CALL(T, V): V channels per lane.  Two for 16-bit types, so that a wave reads 256 bytes of a row as with one fp32 channel
// (four: 300 us forward instead of 225 on 131072 x 1024 bf16); odd row lengths and strides fall back to one.
#define SCAN_BY_TYPE(dtype, vec, CALL)                                        \
    do {                                                                      \
        if ((dtype) == DVAE_F32) { CALL(float, 1); }                          \
        else if ((dtype) == DVAE_BF16) {                                      \
            if ((vec) == 2) { CALL(__bf16, 2); } else { CALL(__bf16, 1); }    \
        } else {                                                              \
            if ((vec) == 2) { CALL(_Float16, 2); } else { CALL(_Float16, 1); } \
        }                                                                     \
    } while (0)

// workgroups that look for sequences without rows
static long scan_empty_blocks(const ScanParams& p, const float* to) {
    return to && p.q.S > 0 && (p.q.off || p.q.len == 0) ? (p.q.S + 3) / 4 : 0;
}

// the launches of a pass: one workgroup per tile and slab, and those that look for sequences without rows beside them or, with
// several tiles, in the launch before
static int scan_grid(const char* who, const ScanParams& p, const ScanWs& L, int threads, const float* to, dim3& grid) {
    const long empty = scan_empty_blocks(p, to), blocks = L.tiles * p.slabs + (L.tiles == 1 ? empty : 0);
    DVAE_REQUIRE(grid_fits(blocks, threads) && grid_fits(FILL_BLOCKS + empty, 256), "%s: %lld rows of %d channels in %lld sequences are too many", who,
                 (long long)p.q.N, p.D, (long long)p.q.S);
    grid = dim3((unsigned)blocks);
    return DVAE_OK;
}

static int scan_begin(ScanParams& p, void* ws, const ScanWs& L, const float* from, float* to, hipStream_t s) {
    p.words = (unsigned long long*)((char*)ws + L.words);
    if (L.tiles == 1) return DVAE_OK;
    p.ticket = (unsigned*)ws;
    const long pairs = (L.tiles * p.D + 1) / 2;
    const int fill = L.tiles == 0 ? 0 : (int)min((pairs + 255) / 256, FILL_BLOCKS);
    const long blocks = fill + scan_empty_blocks(p, to);
    if (blocks == 0) return DVAE_OK;
    hipLaunchKernelGGL(scan_begin_kernel, dim3((unsigned)blocks), dim3(256), 0, s, (ulonglong2*)p.words, pairs, p.ticket, fill,
                       p.q, from, to, p.D);
    DVAE_LAUNCH_CHECK();
    return DVAE_OK;
}

}  // namespace dvae

extern "C" int64_t dvae_scan_state_floats(int64_t rows, int32_t D) {
    using namespace dvae;
    DVAE_TRY(scan_check("scan_state_floats", rows, 1, nullptr, 0, D, DVAE_F32));
    return scan_ws(rows, D, TRB).states;
}
extern "C" int64_t dvae_scan_ws_bytes(int64_t rows, int32_t D) {
    using namespace dvae;
    DVAE_TRY(scan_check("scan_ws_bytes", rows, 1, nullptr, 0, D, DVAE_F32));
    return scan_ws(rows, D, TRB).bytes;
}

extern "C" int dvae_scan_fwd(const void* gate, int64_t ld_gate, const void* x, int64_t ld_x, const void* off, int32_t off_i64,
                             const float* h0, void* h, float* last, float* states, void* ws, int64_t rows, int64_t seqs,
                             int32_t D, int32_t dtype, void* stream) {
    using namespace dvae;
    DVAE_TRY(scan_check("scan_fwd", rows, seqs, off, ld_gate > ld_x ? ld_gate : ld_x, D, dtype));
    DVAE_REQUIRE((ld_gate == 0 || ld_gate >= D) && (ld_x == 0 || ld_x >= D), "scan_fwd: a row stride is below %d channels", D);
    DVAE_REQUIRE(rows == 0 || (gate && x && h && ws), "scan_fwd: null pointer");
    DVAE_REQUIRE(seqs == 0 || last, "scan_fwd: null pointer");
    DVAE_REQUIRE((uintptr_t)ws % 16 == 0, "scan_fwd: the workspace must be 16-byte aligned");
    hipStream_t s = (hipStream_t)stream;
    const ScanWs L = scan_ws(rows, D, TRF);
    const int vec = widest(elem_size(dtype), 4, {(int64_t)D, ld_gate, ld_x}, {gate, x, (const void*)h});
    ScanParams p = {};
    p.gate = gate; p.x = x; p.ld_gate = ld_gate; p.ld_x = ld_x; p.h = h; p.h0 = h0; p.last = last; p.states = states;
    p.q = {off, off_i64, seqs, seqs > 0 ? rows / seqs : 0, rows};
    p.D = D; p.slabs = cdiv(D, 64 * vec);
    dim3 grid;
    DVAE_TRY(scan_grid("scan_fwd", p, L, TRF / RW * 64, last, grid));
    DVAE_TRY(scan_begin(p, ws, L, h0, last, s));
    if (rows == 0) return DVAE_OK;
#define SCAN_FWD(T, V) hipLaunchKernelGGL((scan_fwd_kernel<T, V>), grid, dim3(TRF / RW * 64), 0, s, p)
    SCAN_BY_TYPE(dtype, vec, SCAN_FWD);
#undef SCAN_FWD
    DVAE_LAUNCH_CHECK();
    return DVAE_OK;
}

extern "C" int dvae_scan_bwd(const void* gate, int64_t ld_gate, const void* x, int64_t ld_x, const void* off, int32_t off_i64,
                             const float* h0, const float* states, const void* dh, int64_t ld_dh, const float* dlast, void* dgate,
                             void* dx, float* dh0, void* ws, int64_t rows, int64_t seqs, int32_t D, int32_t dtype, void* stream) {
    using namespace dvae;
    const int64_t ld_in = ld_gate > ld_x ? ld_gate : ld_x;
    DVAE_TRY(scan_check("scan_bwd", rows, seqs, off, ld_in > ld_dh ? ld_in : ld_dh, D, dtype));
    DVAE_REQUIRE((ld_gate == 0 || ld_gate >= D) && (ld_x == 0 || ld_x >= D) && (ld_dh == 0 || ld_dh >= D),
                 "scan_bwd: a row stride is below %d channels", D);
    DVAE_REQUIRE(rows == 0 || (gate && x && states && dgate && dx && ws), "scan_bwd: null pointer");
    DVAE_REQUIRE((uintptr_t)ws % 16 == 0, "scan_bwd: the workspace must be 16-byte aligned");
    hipStream_t s = (hipStream_t)stream;
    const ScanWs L = scan_ws(rows, D, TRB);
    const int vec = widest(elem_size(dtype), 4, {(int64_t)D, ld_gate, ld_x, dh ? ld_dh : 0},
                           {gate, x, dh, (const void*)dgate, (const void*)dx});
    ScanParams p = {};
    p.gate = gate; p.x = x; p.dh = dh; p.ld_gate = ld_gate; p.ld_x = ld_x; p.ld_dh = ld_dh;
    p.dgate = dgate; p.dx = dx; p.h0 = h0; p.dlast = dlast; p.dh0 = dh0; p.states = const_cast<float*>(states);
    p.q = {off, off_i64, seqs, seqs > 0 ? rows / seqs : 0, rows};
    p.D = D; p.slabs = cdiv(D, 64 * vec);
    dim3 grid;
    DVAE_TRY(scan_grid("scan_bwd", p, L, TRB / RW * 64, dh0, grid));
    DVAE_TRY(scan_begin(p, ws, L, dlast, dh0, s));
    if (rows == 0) return DVAE_OK;
#define SCAN_BWD(T, V) hipLaunchKernelGGL((scan_bwd_kernel<T, V>), grid, dim3(TRB / RW * 64), 0, s, p)
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
    // (every row reads all slots, to find the rows that share its own)
    DVAE_REQUIRE(!slots || rows <= 65536, "scan_step: %d rows with slots; at most 65536 are supported", rows);
    DVAE_REQUIRE(slots || rows <= pool, "scan_step: %d rows, but a pool of %lld states", rows, (long long)pool);
    if (rows == 0) return DVAE_OK;
    DVAE_REQUIRE(gate && x && h && (state || pool == 0), "scan_step: null pointer");
    const int vec = widest(elem_size(dtype), 16, {(int64_t)D, ld_gate, ld_x}, {gate, x, (const void*)h});
    const int slabs = cdiv(D, 64 * vec);
    const long units = (long)rows * slabs;
    DVAE_REQUIRE(grid_fits((units + 3) / 4, 256), "scan_step: %d rows of %d channels are too many", rows, D);
    const dim3 grid((unsigned)((units + 3) / 4));
#define SCAN_STEP_BY(T, V, I)                                                                                                   \
    hipLaunchKernelGGL((scan_step_kernel<T, V, I>), grid, dim3(256), 0, (hipStream_t)stream, (const T*)gate, (long)ld_gate,       \
                       (const T*)x, (long)ld_x, state, (long)ld_state, (long)pool, (const I*)slots, (T*)h, rows, D, slabs)
#define SCAN_STEP(T, V) \
    if (slots_i64) SCAN_STEP_BY(T, V, int64_t); else SCAN_STEP_BY(T, V, int32_t)
    DVAE_BY_TYPE(dtype, vec, SCAN_STEP);
#undef SCAN_STEP
#undef SCAN_STEP_BY
    DVAE_LAUNCH_CHECK();
    return DVAE_OK;
}
