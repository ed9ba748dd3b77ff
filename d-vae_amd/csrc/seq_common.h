// Shared by the sequence operators (embed.hip, scan.hip): element types, vector accesses and their widest legal width.
#pragma once
#include "common.h"
#include "dvae_hip.h"

namespace dvae {

// V consecutive elements of T as one access (V * sizeof(T) <= 16 bytes, aligned to that)
template <typename T, int V> struct alignas(sizeof(T) * V) Pack { T e[V]; };

// the access itself as one integer vector (hipcc otherwise splits a constant pack into stores of its elements)
template <int BYTES> struct Word;
template <> struct Word<2> { typedef unsigned short type; };
template <> struct Word<4> { typedef unsigned type; };
template <> struct Word<8> { typedef unsigned type __attribute__((ext_vector_type(2))); };
template <> struct Word<16> { typedef unsigned type __attribute__((ext_vector_type(4))); };
template <typename T, int V> __device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
    typedef typename Word<sizeof(T) * V>::type W;
    return __builtin_bit_cast(Pack<T, V>, *reinterpret_cast<const W*>(p));
}
template <typename T, int V> __device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& v) {
    typedef typename Word<sizeof(T) * V>::type W;
    *reinterpret_cast<W*>(p) = __builtin_bit_cast(W, v);
}
// one rounding, to nearest even
template <typename T, int V> __device__ __forceinline__ void store_floats(T* p, const float (&f)[V]) {
    Pack<T, V> o;
#pragma unroll
    for (int i = 0; i < V; ++i) o.e[i] = (T)f[i];
    store_pack<T, V>(p, o);
}

// The value is in registers here, and nothing computed from it before is reused behind: keeps a load from being sunk behind
// a branch, and what can be recomputed cheaply from being kept in registers across a long section.
template <typename T, int V> __device__ __forceinline__ void hold(Pack<T, V>& v) {
    if constexpr (sizeof(v) >= 4) {
        unsigned w[sizeof(v) / 4];
        __builtin_memcpy(w, &v, sizeof(v));
#pragma unroll
        for (unsigned i = 0; i < sizeof(v) / 4; ++i) asm volatile("" : "+v"(w[i]));
        __builtin_memcpy(&v, w, sizeof(v));
    } else {
        unsigned short w;
        __builtin_memcpy(&w, &v, 2);
        asm volatile("" : "+v"(w));
        __builtin_memcpy(&v, &w, 2);
    }
}
__device__ __forceinline__ void hold(float& v) { asm volatile("" : "+v"(v)); }

static inline int elem_size(int dtype) { return dtype == DVAE_F32 ? 4 : 2; }
static inline bool known_dtype(int dtype) { return dtype == DVAE_F32 || dtype == DVAE_BF16 || dtype == DVAE_F16; }

// the runtime takes less than 2^32 threads along a grid
static inline bool grid_fits(int64_t blocks, int threads) { return blocks * threads < (1LL << 32); }

// The widest vector (in elements, at most `bytes` bytes) that divides every listed extent / stride and to which every
// base pointer is aligned.  An odd row length leaves single elements, which a wave still reads as one 128- or 256-byte run.
template <size_t NE, size_t NP>
static inline int widest(int es, int bytes, const int64_t (&extents)[NE], const void* const (&ptrs)[NP]) {
    for (int v = bytes / es; v > 1; v /= 2) {
        bool ok = true;
        for (int64_t x : extents) ok = ok && x % v == 0;
        for (const void* p : ptrs) ok = ok && (uintptr_t)p % (uintptr_t)(v * es) == 0;
        if (ok) return v;
    }
    return 1;
}

// CALL(T, V) for the element type and vector width picked at run time
#define DVAE_BY_TYPE(dtype, vec, CALL)                                        \
    do {                                                                      \
        if ((dtype) == DVAE_F32) {                                            \
            if ((vec) >= 4) { CALL(float, 4); }                               \
            else if ((vec) == 2) { CALL(float, 2); }                          \
            else { CALL(float, 1); }                                          \
        } else if ((dtype) == DVAE_BF16) {                                    \
            if ((vec) >= 8) { CALL(__bf16, 8); }                              \
            else if ((vec) == 4) { CALL(__bf16, 4); }                         \
            else if ((vec) == 2) { CALL(__bf16, 2); }                         \
            else { CALL(__bf16, 1); }                                         \
        } else {                                                              \
            if ((vec) >= 8) { CALL(_Float16, 8); }                            \
            else if ((vec) == 4) { CALL(_Float16, 4); }                       \
            else if ((vec) == 2) { CALL(_Float16, 2); }                       \
            else { CALL(_Float16, 1); }                                       \
        }                                                                     \
    } while (0)

}  // namespace dvae
