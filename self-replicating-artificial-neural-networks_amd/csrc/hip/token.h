// Shared by the token operators (token_score.hip, token_distill.hip): rows of logits in registers, reductions, launch shapes.
//
// A row is V logits x (fp32, bf16 or fp16) at temperature T; c = log2(e) / T.  With m = max x and mc = m c rounded to fp32,
//   d_v = fma(x_v, c, -mc),  e_v = exp2(d_v),  dmax = fma(m, c, -mc)     (dmax: what the rounding of mc left, |mc| 2^-24)
// every d_v is shifted by the same dmax, so it is taken back once a row instead of paying a subtraction an element.  The
// elements equal to m are counted (n) and left out of the sums: of a row that is nearly sure of one token the rest
//   S = sum_{x_v < m} e_v 2^-dmax
// keeps its digits (1 + S would not), and ln sum = ln(n + S) is log1p(S) for n = 1.  All sums are fp32 over at most 128
// terms a thread, then a fixed tree over lanes and waves (no atomics: the same bits on every run); the distillation loss, a
// small difference of large terms, takes its logarithms and its K terms in fp64.
//
// Rows whose elements are all -inf have no distribution: S = n = 0, flagged by l2S = +inf, which makes every q_v = 0.
// A NaN or +inf logit makes the row's sums NaN.
#pragma once
#include "common.h"
#include "serann_hip.h"
#include <stdexcept>

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 f16_t;

constexpr int TOK_MAX_K = 128;        // top alternatives a row
constexpr int64_t TOK_MAX_V = 1000000;
constexpr int TOK_MAX_SEG = 62;       // segments a row is cut into at most: 10^6 fp32 logits in 64 KB pieces; a lane each to join
constexpr int TOK_NARROW_V = 512;     // rows of up to 64 x 8 elements: a group of 8-64 lanes a row, no LDS reduction

// Rows of a [n0][n1][V] tensor with strides s0, s1 (elements) and unit stride inside a row; row r = (r / n1, r % n1)
struct TokRows {
    int64_t x, rows, n1, s0, s1;
    int64_t u0;           // first unit of this launch (tok_launch)
    int V;
    float c, inv_t;       // log2(e) / T, 1 / T
    double dinv_t;
};

template <typename T> struct TokElem;
template <> struct TokElem<float> {
    static constexpr int VEC = 4;
    static constexpr uint32_t NEG_INF = 0xff800000u;
    static __device__ __forceinline__ float get(const u32x4_t& v, int e) { return __uint_as_float(v[e]); }
    static __device__ __forceinline__ float one(float v) { return v; }
    static __device__ __forceinline__ u32x4_t pack(const float* f) {
        return u32x4_t{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
    }
    static __device__ __forceinline__ float put(float f) { return f; }
};
template <> struct TokElem<bf16_t> {
    static constexpr int VEC = 8;
    static constexpr uint32_t NEG_INF = 0xff80ff80u;
    static __device__ __forceinline__ float get(const u32x4_t& v, int e) {
        return __uint_as_float((e & 1) ? (v[e >> 1] & 0xffff0000u) : (v[e >> 1] << 16));
    }
    static __device__ __forceinline__ float one(bf16_t v) { return bf2f(v); }
    static __device__ __forceinline__ u32x4_t pack(const float* f) {
        return u32x4_t{f2bf2(f[0], f[1]), f2bf2(f[2], f[3]), f2bf2(f[4], f[5]), f2bf2(f[6], f[7])};
    }
    static __device__ __forceinline__ bf16_t put(float f) { return f2bf(f); }
};
template <> struct TokElem<f16_t> {
    static constexpr int VEC = 8;
    static constexpr uint32_t NEG_INF = 0xfc00fc00u;
    static __device__ __forceinline__ float get(const u32x4_t& v, int e) {
        return (float)__builtin_bit_cast(f16_t, (uint16_t)(v[e >> 1] >> ((e & 1) * 16)));
    }
    static __device__ __forceinline__ float one(f16_t v) { return (float)v; }
    static __device__ __forceinline__ u32x4_t pack(const float* f) {
        u32x4_t o;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            o[i] = (uint32_t)__builtin_bit_cast(uint16_t, (f16_t)f[2 * i]) |
                   ((uint32_t)__builtin_bit_cast(uint16_t, (f16_t)f[2 * i + 1]) << 16);
        return o;
    }
    static __device__ __forceinline__ f16_t put(float f) { return (f16_t)f; }
};

// 16 bytes at any element's address: a row starts where its stride puts it (odd V), and gfx950 takes unaligned vectors.
// Addresses that come as integers are told to be global memory (a flat access would wait for LDS too).
#define TOK_GLOBAL __attribute__((address_space(1)))
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
template <typename T> using tok_in = const TOK_GLOBAL T*;
template <typename T> using tok_out = TOK_GLOBAL T*;
template <typename T> __device__ __forceinline__ u32x4_t tok_ld16(tok_in<T> p) {
    return *(tok_in<u32x4_any>)p;
}
template <typename T> __device__ __forceinline__ void tok_st16(tok_out<T> p, u32x4_t v) { *(tok_out<u32x4_any>)p = v; }

// max without the canonicalising multiplies that fmaxf brings for signalling NaNs; a NaN operand is passed over (it comes
// back through the sums)
__device__ __forceinline__ float tok_max(float a, float b) {
    float r;
    asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ float tok_max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
__device__ __forceinline__ float tok_exp2(float d) { return __builtin_amdgcn_exp2f(d); }

template <int CTRL> __device__ __forceinline__ float tok_dpp(float v) {
    const int i = __builtin_bit_cast(int, v);
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, CTRL, 0xf, 0xf, false));
}
template <int CTRL> __device__ __forceinline__ uint32_t tok_dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false);
}
template <int CTRL> __device__ __forceinline__ uint64_t tok_dpp(uint64_t v) {
    return (uint64_t)tok_dpp<CTRL>((uint32_t)v) | ((uint64_t)tok_dpp<CTRL>((uint32_t)(v >> 32)) << 32);
}
template <int CTRL> __device__ __forceinline__ double tok_dpp(double v) {
    return __builtin_bit_cast(double, tok_dpp<CTRL>(__builtin_bit_cast(uint64_t, v)));
}
struct TokMax { static __device__ __forceinline__ float f(float a, float b) { return tok_max(a, b); } };
struct TokMin {
    static __device__ __forceinline__ float f(float a, float b) { return fminf(a, b); }
    static __device__ __forceinline__ uint64_t f(uint64_t a, uint64_t b) { return a < b ? a : b; }
};
struct TokSum {
    static __device__ __forceinline__ float f(float a, float b) { return a + b; }
    static __device__ __forceinline__ double f(double a, double b) { return a + b; }
    static __device__ __forceinline__ uint32_t f(uint32_t a, uint32_t b) { return a + b; }
};
struct TokTop {
    static __device__ __forceinline__ uint32_t f(uint32_t a, uint32_t b) { return a > b ? a : b; }
    static __device__ __forceinline__ uint64_t f(uint64_t a, uint64_t b) { return a > b ? a : b; }
    static __device__ __forceinline__ double f(double a, double b) { return a > b ? a : b; }
};
// (a, b) of lanes 16 (32) apart: the even row of 16 lanes (the lower half) of v in every lane, and the odd row (upper half)
template <int D> __device__ __forceinline__ void tok_halves(uint32_t v, uint32_t& a, uint32_t& b) {
    static_assert(D == 16 || D == 32, "rows or halves");
    if constexpr (D == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        a = r[0];
        b = r[1];
    } else {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        a = r[0];
        b = r[1];
    }
}
template <int D, typename OP, typename V> __device__ __forceinline__ V tok_across(V v) {
    if constexpr (sizeof(V) == 4) {
        uint32_t a, b;
        tok_halves<D>(__builtin_bit_cast(uint32_t, v), a, b);
        return OP::f(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b));
    } else {
        const uint64_t w = __builtin_bit_cast(uint64_t, v);
        uint32_t al, bl, ah, bh;
        tok_halves<D>((uint32_t)w, al, bl);
        tok_halves<D>((uint32_t)(w >> 32), ah, bh);
        return OP::f(__builtin_bit_cast(V, (uint64_t)ah << 32 | al), __builtin_bit_cast(V, (uint64_t)bh << 32 | bl));
    }
}
// Reduction over aligned groups of G lanes, every lane gets the result: lanes 1 and 2 apart (quad_perm), then the mirrored
// half row and row (their quads / halves are uniform by then), then across rows of 16: all on the vector ALU, no LDS trip
template <int G, typename OP, typename V> __device__ __forceinline__ V tok_group(V v) {
    if constexpr (G > 1) v = OP::f(v, tok_dpp<0xB1>(v));
    if constexpr (G > 2) v = OP::f(v, tok_dpp<0x4E>(v));
    if constexpr (G > 4) v = OP::f(v, tok_dpp<0x141>(v));
    if constexpr (G > 8) v = OP::f(v, tok_dpp<0x140>(v));
    if constexpr (G > 16) v = tok_across<16, OP>(v);
    if constexpr (G > 32) v = tok_across<32, OP>(v);
    return v;
}

// (value, index) as one unsigned key, larger = ranked first: the float's bits in their order, then the lowest index.
// +0.0 joins -0 and +0, which are equal values.
__device__ __forceinline__ uint32_t tok_order(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float tok_unorder(uint32_t o) {
    return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t tok_key(float x, int i) {
    return ((uint64_t)tok_order(x) << 32) | (uint32_t)~(uint32_t)i;
}
__device__ __forceinline__ int tok_key_index(uint64_t k) { return (int)~(uint32_t)k; }
__device__ __forceinline__ float tok_key_value(uint64_t k) { return tok_unorder((uint32_t)(k >> 32)); }

// Ranks the n distinct keys of an LDS list (16-byte aligned) by counting the larger ones, 8 lanes a key, two keys a read: f(rank,
// key) for ranks below k, from one lane.  n is the same in every thread; NT threads call.
template <int NT, typename F> __device__ __forceinline__ void tok_count_ranks(const uint64_t* keys, int n, int k, const F& f) {
    const int tid = threadIdx.x, l = tid & 7;
    const ulonglong2* two = reinterpret_cast<const ulonglong2*>(keys);
    for (int i0 = 0; i0 < n; i0 += NT / 8) {
        const int i = i0 + (tid >> 3);
        const uint64_t key = i < n ? keys[i] : 0;
        uint32_t c = 0;
        int j = l;
        for (; j + 24 < n / 2; j += 32) {
            const ulonglong2 a = two[j], b = two[j + 8], d = two[j + 16], e = two[j + 24];
            c += (a.x > key) + (a.y > key) + (b.x > key) + (b.y > key) + (d.x > key) + (d.y > key) + (e.x > key) + (e.y > key);
        }
        for (; j < n / 2; j += 8) {
            const ulonglong2 a = two[j];
            c += (a.x > key) + (a.y > key);
        }
        if ((n & 1) && l == 0) c += keys[n - 1] > key;
        c = tok_group<8, TokSum>(c);
        if (l == 0 && i < n && (int)c < k) f((int)c, key);
    }
}

// Sorting, largest first.  Within a lane: networks of 1, 2, 4 or 8 keys (Batcher's odd-even merge sort).
template <typename K> __device__ __forceinline__ void tok_order2(K& a, K& b) {
    const K hi = a > b ? a : b, lo = a > b ? b : a;
    a = hi;
    b = lo;
}
template <int E, typename K> __device__ __forceinline__ void tok_sort_lane(K* h) {
    static_assert(E == 1 || E == 2 || E == 4 || E == 8, "keys a lane");
#pragma unroll
    for (int e = 0; e + 1 < E; e += 2) tok_order2(h[e], h[e + 1]);
#pragma unroll
    for (int e = 0; e + 3 < E; e += 4) {
        tok_order2(h[e], h[e + 2]);
        tok_order2(h[e + 1], h[e + 3]);
        tok_order2(h[e + 1], h[e + 2]);
    }
    if constexpr (E == 8) {
        tok_order2(h[0], h[4]); tok_order2(h[1], h[5]); tok_order2(h[2], h[6]); tok_order2(h[3], h[7]);
        tok_order2(h[2], h[4]); tok_order2(h[3], h[5]);
        tok_order2(h[1], h[2]); tok_order2(h[3], h[4]); tok_order2(h[5], h[6]);
    }
}
// v of the lane whose number differs in the bits of D, inside a group of lanes
template <int D> __device__ __forceinline__ uint32_t tok_other(uint32_t v, int lane) {
    uint32_t a, b;
    tok_halves<D>(v, a, b);
    return (lane & D) ? a : b;
}
template <int D> __device__ __forceinline__ uint64_t tok_other(uint64_t v, int lane) {
    return (uint64_t)tok_other<D>((uint32_t)v, lane) | (uint64_t)tok_other<D>((uint32_t)(v >> 32), lane) << 32;
}
template <int D, typename K> __device__ __forceinline__ K tok_xor(K v, int lane) {
    if constexpr (D >= 32) {
        return tok_other<32>(tok_xor<D & 31>(v, lane), lane);
    } else if constexpr (D >= 16) {
        return tok_other<16>(tok_xor<D & 15>(v, lane), lane);
    } else if constexpr (D == 0) {
        return v;
    } else if constexpr (D == 4) {
        return tok_dpp<0x1B>(tok_dpp<0x141>(v));             // 7, then 3
    } else {
        static_assert(D == 1 || D == 2 || D == 3 || D == 7 || D == 8 || D == 15, "one DPP move");
        return tok_dpp<D == 1 ? 0xB1 : D == 2 ? 0x4E : D == 3 ? 0x1B : D == 7 ? 0x141 : D == 8 ? 0x128 : 0x140>(v);
    }
}
// Every lane's E keys against those of the lane D apart: where `low`, the larger keys stay.  FLIP: key e meets key E - 1 - e
template <int D, int E, bool FLIP, typename K> __device__ __forceinline__ void tok_exchange(K* h, int lane, bool low) {
    K o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = tok_xor<D>(h[FLIP ? E - 1 - e : e], lane);
#pragma unroll
    for (int e = 0; e < E; ++e) h[e] = (h[e] > o[e]) == low ? h[e] : o[e];
}
template <int D, int E, typename K> __device__ __forceinline__ void tok_clean(K* h, int lane) {
    if constexpr (D >= 1) {
        tok_exchange<D, E, false>(h, lane, !(lane & D));
        tok_clean<D / 2, E>(h, lane);
    } else {
#pragma unroll
        for (int d = E / 2; d >= 1; d /= 2)
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (!(e & d)) tok_order2(h[e], h[e + d]);
    }
}
// Bitonic merges of the sorted E keys of G lanes: then lane g has the ranks E g to E g + E - 1.  Two sorted runs of L lanes meet
// head against tail (lanes 2 L - 1 apart), which leaves the larger half in the lower lanes.  lane: the number in the group
template <int G, int E, int L = 1, typename K> __device__ __forceinline__ void tok_sort_group(K* h, int lane) {
    if constexpr (L < G) {
        tok_exchange<2 * L - 1, E, true>(h, lane, !(lane & L));
        tok_clean<L / 2, E>(h, lane);
        tok_sort_group<G, E, 2 * L>(h, lane);
    }
}
// The largest k of the n <= 64 E keys of an LDS list, sorted by one wave: f(rank, key), each from one lane
template <int E, typename F> __device__ __forceinline__ void tok_sort_list(const uint64_t* keys, int n, int k, const F& f) {
    const int lane = threadIdx.x & 63;
    uint64_t h[E];
#pragma unroll
    for (int e = 0; e < E; ++e) h[e] = e * 64 + lane < n ? keys[e * 64 + lane] : 0;
    tok_sort_lane<E>(h);
    tok_sort_group<64, E>(h, lane);
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (lane * E + e < min(n, k)) f(lane * E + e, h[e]);
}

// The k largest of a list by counting or, where it is long, by the first wave's sort: one wave a row sorts from 17 keys on (120,000
// rows of 1,000 fp32 logits, k = 64: 234 us, counting 337; k = 4: 160 and 146), blocks of more waves from 97 on (5,000 rows of
// 6,000 fp32 logits, k = 100: 41 us, counting 50; k = 20: no difference; 48 of 128,001 bf16, k = 128, some 300 keys: 18 and 24).
template <int NT, typename F> __device__ __forceinline__ void tok_rank(const uint64_t* keys, int n, int k, const F& f) {
    if (n > (NT == 64 ? 16 : 96) && n <= (NT == 64 ? 256 : 512)) {
        if (NT > 64 && threadIdx.x >= 64) return;
        if (NT == 64 && n <= 64) tok_sort_list<1>(keys, n, k, f);
        else if (n <= 128) tok_sort_list<2>(keys, n, k, f);
        else if (n <= 256) tok_sort_list<4>(keys, n, k, f);
        else if constexpr (NT > 64) tok_sort_list<8>(keys, n, k, f);
    } else {
        tok_count_ranks<NT>(keys, n, k, f);
    }
}

template <typename T> __device__ __forceinline__ tok_in<T> tok_row(const TokRows& r, int64_t row) {
    const int64_t i0 = r.n1 == r.rows ? 0 : (int64_t)((uint32_t)row / (uint32_t)r.n1);      // fewer than 2^31 rows
    return (tok_in<T>)r.x + i0 * r.s0 + (row - i0 * r.n1) * r.s1;
}
__device__ __forceinline__ int64_t tok_int(int64_t base, int is64, int64_t i) {
    return is64 ? ((tok_in<int64_t>)base)[i] : (int64_t)((tok_in<int32_t>)base)[i];
}

// A row's exponents, d = fma(x, c, -mc).  dmax is up to half a step of mc: 2^6 below |m| c = 2^31, so that 2^-dmax stays finite,
// and any number of octaves above it.  But from 2^31 on two different fp32 logits lie at least 2^31 2^-24 = 128 octaves apart, so
// only those equal to m count there: everything else gets -inf, and dmax is 0.
struct TokRef {
    float c, mc, dmax, meq;      // meq: the value of the elements to count (a NaN, equal to nothing, in a row of -inf)
};
__device__ __forceinline__ TokRef tok_ref(float m, float c) {
    const bool none = m == -INFINITY, big = !none && fabsf(m) * c >= 2147483648.f;
    TokRef r;
    r.c = big ? 1e-30f : c;
    r.mc = none ? 0.f : big ? INFINITY : m * c;
    r.dmax = none || big ? 0.f : __builtin_fmaf(m, c, -r.mc);
    r.meq = none ? NAN : m;
    return r;
}

// ln(n + S) of a row's sums (n elements at the maximum, S over the others)
__device__ __forceinline__ float tok_ln(float n, float S) { return n == 1.f ? log1pf(S) : logf(n + S); }

// lanes below this one whose bit is set
__device__ __forceinline__ int tok_below(uint64_t mask) {
    return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}
// Vectors that need a look at each element (one with the maximum, with candidates of the top k, with listed tokens) go, data
// and place, to their wave's list in LDS, out of the unrolled pass.  Slots are counted by ballots: no atomics, one order.
// What is summed is summed by the thread that pushed the vector, along its own chain of slots.
template <int CAP> struct TokSpecial {
    u32x4_t data[CAP];
    int at[CAP], next[CAP];      // vector of the segment (bit 31: to be summed), the thread's slot before this one
    // all lanes of the wave; n: the list's length so far (over CAP: it did not fit)
    __device__ __forceinline__ void push(bool hit, const u32x4_t& v, int where, bool sum, int& chain, int& n) {
        const uint64_t mask = __ballot(hit);
        if (mask == 0) return;
        const int i = n + tok_below(mask);
        if (hit && i < CAP) {
            data[i] = v;
            at[i] = where | (sum ? (int)0x80000000 : 0);
            next[i] = chain;
            chain = i;
        }
        n += (int)__popcll(mask);
    }
    __device__ __forceinline__ int vec(int slot) const { return at[slot] & 0x7fffffff; }
    template <typename T> __device__ __forceinline__ float get(int slot, int e) const {
        return TokElem<T>::one(reinterpret_cast<const T*>(&data[slot])[e]);
    }
};

// A lower bound of the k-th largest of the wave's lanes' values (1 <= k <= 64): at least k of them are at or above it, seldom
// many more.  Bisection on the value, counted by ballots; -inf where fewer than k lanes have more.
__device__ __forceinline__ float tok_kth_bound(float v, int k) {
    const float hi0 = tok_group<64, TokMax>(v);
    float lo = tok_group<64, TokMin>(v > -INFINITY ? v : INFINITY), hi = hi0;
    if (k == 1) return hi0;
    if ((int)__popcll(__ballot(v >= lo)) < k || !(hi < INFINITY)) return -INFINITY;
    for (int it = 0; it < 10; ++it) {
        const float mid = 0.5f * lo + 0.5f * hi;
        const int c = (int)__popcll(__ballot(v >= mid));
        if (c >= k) {
            lo = mid;
            if (c <= k + (k >> 2) + 1) break;
        } else {
            hi = mid;
        }
    }
    return lo;
}

// A segment of a row in registers: NV 16-byte vectors a thread and one of the < VEC last elements of the row.  Vector
// i * NT + tid of the segment is r[i]; vm[i] its maximum.
template <typename T, int NT, int NV> struct TokSeg {
    static constexpr int VEC = TokElem<T>::VEC;
    u32x4_t r[NV];
    float vm[NV];
    float xt;
    int nv;             // full vectors of the segment
    __device__ __forceinline__ void load(tok_in<T> x, int nvec, int ntail) {
        const int tid = threadIdx.x;
        asm("" : "+s"(nvec));                               // masks made here and now, not kept from row to row
        nv = nvec;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            tok_in<T> p = x + i * NT * VEC;                 // uniform; the thread's part of the address is one 32-bit offset
            if ((i + 1) * NT <= nvec) {
                r[i] = tok_ld16<T>((tok_in<T>)((tok_in<char>)p + (uint32_t)tid * 16u));
            } else {
                r[i] = u32x4_t{TokElem<T>::NEG_INF, TokElem<T>::NEG_INF, TokElem<T>::NEG_INF, TokElem<T>::NEG_INF};
                if (i * NT + tid < nvec) r[i] = tok_ld16<T>((tok_in<T>)((tok_in<char>)p + (uint32_t)tid * 16u));
            }
        }
        xt = -INFINITY;
        if (tid < ntail) xt = TokElem<T>::one(x[nvec * VEC + tid]);
    }
    __device__ __forceinline__ float max_of() {
        float m = xt;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float a = tok_max3(TokElem<T>::get(r[i], 0), TokElem<T>::get(r[i], 1), TokElem<T>::get(r[i], 2));
            if constexpr (VEC == 4) {
                a = tok_max(a, TokElem<T>::get(r[i], 3));
            } else {
                a = tok_max3(a, TokElem<T>::get(r[i], 3), TokElem<T>::get(r[i], 4));
                a = tok_max3(a, TokElem<T>::get(r[i], 5), TokElem<T>::get(r[i], 6));
                a = tok_max(a, TokElem<T>::get(r[i], 7));
            }
            vm[i] = a;
            m = tok_max(m, a);
        }
        forget();
        return m;
    }
    // the wave's elements at or above B (B > -inf)
    __device__ __forceinline__ int count(float B) const {
        int c = (int)__popcll(__ballot(xt >= B));
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (i * NT < nv) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) c += (int)__popcll(__ballot(TokElem<T>::get(r[i], e) >= B));
            }
        return c;
    }
    // The next pass unpacks the elements again: kept from pass to pass they would take a register each, not half of one
    __device__ __forceinline__ void forget() {
#pragma unroll
        for (int i = 0; i < NV; ++i) asm("" : "+v"(r[i]));
    }
};

// Narrow rows: the 8 elements from e0 on that a lane holds, -inf behind the row's end
template <typename T> __device__ __forceinline__ void tok_narrow_load(tok_in<T> x, int V, int e0, bool live, float* f) {
    constexpr int VEC = TokElem<T>::VEC;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = -INFINITY;
    if (!live) return;
    if (e0 + 8 <= V) {
#pragma unroll
        for (int h = 0; h < 8 / VEC; ++h) {
            const u32x4_t v = tok_ld16<T>(x + e0 + h * VEC);
#pragma unroll
            for (int e = 0; e < VEC; ++e) f[h * VEC + e] = TokElem<T>::get(v, e);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e0 + e < V) f[e] = TokElem<T>::one(x[e0 + e]);
    }
}
template <typename T> __device__ __forceinline__ void tok_narrow_store(tok_out<T> o, int V, int e0, const float* f) {
    constexpr int VEC = TokElem<T>::VEC;
    if (e0 + 8 <= V) {
#pragma unroll
        for (int h = 0; h < 8 / VEC; ++h) tok_st16<T>(o + e0 + h * VEC, TokElem<T>::pack(f + h * VEC));
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e0 + e < V) o[e0 + e] = TokElem<T>::put(f[e]);
    }
}

// Many short rows (up to 64 elements): a wave takes 64 of them, a row a lane -- no reductions between lanes, no idle lanes.
// The rows pass through LDS on the way in and out, so that HBM sees whole lines; a lane's own row there also answers the
// look-ups by token.  LDS holds [64][V] elements; everything is the wave's own, so fences of the wave order it.
__device__ __forceinline__ void tok_wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
// n contiguous elements between global memory and LDS, 16 bytes a lane; all loads of 10 KB (64 rows of 160 bytes) under way at
// once: a wave has no other to wait with
template <typename T> __device__ __forceinline__ void tok_stage_in(tok_in<T> x, T* lds, int n) {
    constexpr int VEC = TokElem<T>::VEC, N = 10;
    const int lane = threadIdx.x, nv = n / VEC;
    u32x4_t* l = reinterpret_cast<u32x4_t*>(lds);
    for (int v0 = 0; v0 < nv; v0 += 64 * N) {
        u32x4_t r[N];
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (v0 + i * 64 + lane < nv) r[i] = tok_ld16<T>(x + (v0 + i * 64 + lane) * VEC);
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (v0 + i * 64 + lane < nv) l[v0 + i * 64 + lane] = r[i];
    }
    for (int e = nv * VEC + lane; e < n; e += 64) lds[e] = x[e];
}
template <typename T> __device__ __forceinline__ void tok_stage_out(const T* lds, tok_out<T> o, int n) {
    constexpr int VEC = TokElem<T>::VEC;
    const int lane = threadIdx.x, nv = n / VEC;
    const u32x4_t* l = reinterpret_cast<const u32x4_t*>(lds);
    for (int v = lane; v < nv; v += 64) tok_st16<T>(o + v * VEC, l[v]);
    for (int e = nv * VEC + lane; e < n; e += 64) o[e] = lds[e];
}
// rows [row0, row0 + n) of the logits to LDS
template <typename T> __device__ __forceinline__ void tok_stage_rows(const TokRows& r, int64_t row0, int n, T* lds) {
    if (r.n1 == r.rows && r.s1 == r.V) {
        tok_stage_in<T>(tok_row<T>(r, row0), lds, n * r.V);
    } else {
        const int lane = threadIdx.x;
        for (int i = 0; i < n; ++i) {
            tok_in<T> x = tok_row<T>(r, row0 + i);
            if (lane < r.V) lds[i * r.V + lane] = x[lane];
        }
    }
    tok_wave_fence();
}
template <typename T> struct TokLane {
    static constexpr int VEC = TokElem<T>::VEC, NVL = 64 / VEC;
    float f[64];
    // the lane's row in LDS; `pad` behind its end
    __device__ __forceinline__ void load(const T* x, int V, float pad) {
        const bool vec = V % VEC == 0;                       // rows start at multiples of 16 bytes
#pragma unroll
        for (int i = 0; i < NVL; ++i) {
            if (i * VEC < V) {                               // uniform
                if (vec) {
                    const u32x4_t v = *reinterpret_cast<const u32x4_t*>(x + i * VEC);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) f[i * VEC + e] = TokElem<T>::get(v, e);
                } else {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        f[i * VEC + e] = pad;
                        if (i * VEC + e < V) f[i * VEC + e] = TokElem<T>::one(x[i * VEC + e]);
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) f[i * VEC + e] = pad;
            }
        }
    }
    __device__ __forceinline__ void store(T* o, int V) const {
        const bool vec = V % VEC == 0;
#pragma unroll
        for (int i = 0; i < NVL; ++i)
            if (i * VEC < V) {
                if (vec) {
                    *reinterpret_cast<u32x4_t*>(o + i * VEC) = TokElem<T>::pack(f + i * VEC);
                } else {
#pragma unroll
                    for (int e = 0; e < VEC; ++e)
                        if (i * VEC + e < V) o[i * VEC + e] = TokElem<T>::put(f[i * VEC + e]);
                }
            }
    }
    // over the elements of the row, VEC at a time (the last chunk's pads among them)
    template <typename F> __device__ __forceinline__ void each(int V, const F& g) {
#pragma unroll
        for (int i = 0; i < NVL; ++i)
            if (i * VEC < V) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) g(i * VEC + e, f[i * VEC + e]);
            }
    }
    __device__ __forceinline__ float max_of(int V, float m) const {
#pragma unroll
        for (int i = 0; i < NVL; ++i)
            if (i * VEC < V) {
#pragma unroll
                for (int e = 0; e < VEC; e += 2) m = tok_max3(m, f[i * VEC + e], f[i * VEC + e + 1]);
            }
        return m;
    }
};

// How a row is taken: NT threads x NV vectors.  Rows of up to `whole` vectors stay one block (two launches cost more than idle
// CUs: one row of 32,000 bf16 logits with 20 alternatives takes 8.1 us whole and 11.1 us in 7 pieces, 32 rows 9.5 and
// 13.7); longer ones are cut into pieces of up to 4096 vectors (64 KB: four blocks a CU, so that one loads while another
// counts; pieces of 8192 make 1,000 rows of 128,001 bf16 logits 57 us instead of 50) and joined by a second launch.
constexpr int TOK_PIECE_VEC = 4096;
static_assert((TOK_MAX_V / 4 + TOK_PIECE_VEC - 1) / TOK_PIECE_VEC <= TOK_MAX_SEG && TOK_MAX_SEG <= 64,
              "the join of the scores gives each segment of a row a lane");
struct TokPlan {
    int nt, nv, nseg, segvec;
};
inline TokPlan tok_plan(int64_t V, int esize, int whole) {
    const int64_t vec = 16 / esize, nvec = V / vec;
    int64_t nseg = nvec <= whole ? 1 : (nvec + TOK_PIECE_VEC - 1) / TOK_PIECE_VEC;
    if (nseg < 1) nseg = 1;
    const int64_t segvec = (nvec + nseg - 1) / nseg;
    nseg = segvec ? (nvec + segvec - 1) / segvec : 1;        // no empty segment
    TokPlan p{0, 0, (int)nseg, (int)segvec};
    static const int shapes[][2] = {{64, 2}, {64, 4}, {64, 8}, {256, 4}, {256, 8}, {256, 16}, {512, 16}, {1024, 16}};
    for (auto& s : shapes)
        if ((int64_t)s[0] * s[1] >= segvec) {
            p.nt = s[0];
            p.nv = s[1];
            break;
        }
    return p;
}
// Launches over `units` of work, a block each: HIP counts a launch's threads in 32 bits, so longer work is several launches.
// (A loop over units inside the kernels would do too, but the compiler then keeps the constants of
// the fp64 functions in registers from unit to unit, up to 60 of them.)
template <typename A, typename... X>
inline void tok_launch(void (*kernel)(A, X...), int64_t units, int nt, size_t lds, hipStream_t s, A a, X... more) {
    const int64_t cap = ((int64_t)1 << 31) / nt;
    for (a.r.u0 = 0; a.r.u0 < units; a.r.u0 += cap) {
        const int64_t n = units - a.r.u0 < cap ? units - a.r.u0 : cap;
        hipLaunchKernelGGL(kernel, dim3((unsigned)n), dim3(nt), lds, s, a, more...);
        SERANN_CHECK(hipGetLastError());
    }
}
inline TokRows tok_rows_of(uint64_t x, int64_t rows, int64_t n1, int64_t s0, int64_t s1, int64_t V, double temperature) {
    // a tensor that only wraps another (functionalisation) has pointer 0: no kernel may read that
    if (rows && !x) throw std::runtime_error("token operators: the logits have no storage");
    if (rows < 0 || V < 1 || V > TOK_MAX_V) throw std::runtime_error("token operators: vocabulary must be in [1, 10^6]");
    if (n1 < 1 || (rows && rows % n1)) throw std::runtime_error("token operators: rows must be a multiple of n1");
    if (!(temperature > 0)) throw std::runtime_error("token operators: temperature must be positive");
    TokRows r;
    r.x = (int64_t)x;
    r.rows = rows;
    r.n1 = n1;
    r.s0 = s0;
    r.s1 = s1;
    r.u0 = 0;
    r.V = (int)V;
    r.c = (float)(1.4426950408889634 / temperature);
    r.inv_t = (float)(1.0 / temperature);
    r.dinv_t = 1.0 / temperature;
    return r;
}
inline int tok_esize(int dtype) { return dtype == 0 ? 4 : 2; }
// lanes a narrow row takes: 8 elements a lane
inline int tok_narrow_lanes(int64_t V) { return V <= 64 ? 8 : V <= 128 ? 16 : V <= 256 ? 32 : 64; }
// A row a lane instead of a row on 8 lanes: where 8 lanes of 8 elements would idle (rows of up to 160 bytes, which also keeps 15
// waves' rows in a CU's LDS) and waves of 64 rows still fill the chip.  A single such wave takes longer (8.4 us with five
// alternatives, 4.9 on 8 lanes); at V = 40 the two meet near 50,000 rows (fp32, 65,536 rows: 9.6 us against 13.3), at V = 64
// in fp32 the 8 lanes stay ahead (179,200 rows: 12.9 us against 17.9 without alternatives).
constexpr int64_t TOK_LANE_ROWS = 65536;
inline bool tok_lane_rows(int64_t V, int esize, int64_t rows) { return V <= 64 && V * esize <= 160 && rows >= TOK_LANE_ROWS; }
