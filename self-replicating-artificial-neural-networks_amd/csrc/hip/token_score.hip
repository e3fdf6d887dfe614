// Log-probabilities of given tokens, with the entropy and the top alternatives of each position, and their backward pass.
//
//   z = x / T, q_v = exp(z_v) / sum exp z;   logprob = ln q_target,   entropy H = -sum q_v ln q_v,
//   top: the k largest x, ties by the lowest index, with their ln q
//   backward: dx_v = ( g_lp ([v = target] - q_v) - g_H q_v (ln q_v + H) ) / T
//
// (token.h has the notation.)  With W = sum_{x_v < m} e_v (d_v - dmax) 2^-dmax:  H = ln(n + S) - ln2 W / (n + S).
//
// Forward, wide rows: a block holds a row (or a segment of one) in registers: one read of HBM, the maximum, then the sums;
// nothing is rescaled and nothing is read twice.  What bounds it: HBM, with ~13 of the ~15 lane operations an element that
// 256 CUs have at 5 TB/s of bf16, so every operation an element counts (one fma to the exponent, v_max3, no canonicalisation).
// Top k: k threads' maxima are k different elements, so the smallest of the per-wave ceil(k / waves)-th largest thread
// maxima is a lower bound of the k-th largest element.  The vectors that reach it go to an LDS list (about 1.5 k of them);
// their elements at or above it are ranked: no data-dependent loop.  Where the lists overflow (thousands of equal values) or fewer
// than k elements are left (masks), the k-th value is found by counting instead (score_select), the row read again from L2.
// Narrow rows (V <= 512, the autoencoder's vocabulary): 8 to 64 lanes a row with 8 elements each; the lane's 8 keys are
// sorted by a network, and k rounds take the best head of the group or, for many alternatives, merges sort the row.
#include "token.h"

struct ScoreArgs {
    TokRows r;
    int64_t y, t0, t1, ignore;   // targets (0: none), their strides
    int y64, k, kj;              // kj: see tok_counted_bound; 0 where k lanes' maxima do
    int nseg, segvec;
    float *lp, *ent;
    int64_t* ids;
    float* top;
    float* stat;                 // for the backward pass: (m, log2 sum, entropy) a row, 0: not wanted
    float4* part;                // nseg > 1: (m, n, S, W) and the sorted keys of each segment
    uint64_t* keys;
};

__device__ __forceinline__ int64_t score_target(const ScoreArgs& a, int64_t row) {
    const int64_t i0 = a.r.n1 == a.r.rows ? 0 : (int64_t)((uint32_t)row / (uint32_t)a.r.n1);
    return tok_int(a.y, a.y64, i0 * a.t0 + (row - i0 * a.r.n1) * a.t1);
}
// Row statistics -> outputs that do not depend on k.  xt: the target's logit (valid_t: the target is inside the vocabulary)
__device__ __forceinline__ float score_finish(const ScoreArgs& a, int64_t row, float m, float n, float S, float W, float xt,
                                              bool valid_t, bool writer) {
    const float lnS = tok_ln(n, S);
    const bool none = n == 0.f && S == 0.f;      // every element -inf (a NaN row has S = NaN)
    if (writer) {
        if (a.lp) a.lp[row] = !valid_t ? NAN : none ? -INFINITY : (xt - m) * a.r.inv_t - lnS;
        const float H = none ? 0.f : lnS - 0.6931471805599453f * (W / (n + S));
        a.ent[row] = H;
        if (a.stat) {
            a.stat[row * 3] = none ? 0.f : m;
            a.stat[row * 3 + 1] = none ? INFINITY : lnS * 1.4426950408889634f;
            a.stat[row * 3 + 2] = H;
        }
    }
    return none ? 0.f : lnS;
}
// lanes = 0: without the alternatives
__device__ __forceinline__ void score_skip(const ScoreArgs& a, int64_t row, int lane, int lanes) {
    if (lane == 0) {
        if (a.lp) a.lp[row] = 0.f;
        a.ent[row] = 0.f;
    }
    for (int j = lane; lanes && j < a.k; j += lanes) {
        a.ids[row * a.k + j] = -1;
        a.top[row * a.k + j] = -INFINITY;
    }
}
__device__ __forceinline__ float score_toplp(const ScoreArgs& a, float x, float m, float lnS) {
    return x == -INFINITY ? -INFINITY + lnS : (x - m) * a.r.inv_t - lnS;
}

// One element's share of the sums
struct ScoreSums {
    float S, W, n;
    __device__ __forceinline__ void add(float x, const TokRef& ref) {
        const float d = __builtin_fmaf(x, ref.c, -ref.mc);
        const bool is = x == ref.meq;
        const float e = is ? 0.f : tok_exp2(d);
        n += is ? 1.f : 0.f;
        S += e;
        W = __builtin_fmaf(e, tok_max(d, -200.f), W);        // -inf: 0 * -200, not 0 * -inf
    }
};

// One wave, many alternatives: k lanes' maxima would be a poor bound (of 64 lanes the lowest one).  A value that some 1.25 k
// elements should reach, were they spread evenly -- the kj-th largest of the lanes' maxima -- is put right by counting the row's
// elements at or above it: k to `cap` of them are looked for, by steps and bisection.  -inf, or more than cap, where 16 counts
// do not find such a value.
template <typename SEG>
__device__ __forceinline__ float tok_counted_bound(const SEG& s, float tm, float m, int k, int kj, int cap) {
    float B = tok_kth_bound(tm, kj), lo = -INFINITY, hi = m;
    if (!(m < INFINITY)) return -INFINITY;
    if (B == -INFINITY) B = tok_group<64, TokMin>(tm > -INFINITY ? tm : m);
    float step = m > B ? m - B : fabsf(m) * 0.0078125f + 1e-6f;
    for (int it = 0; it < 16 && B > -INFINITY; ++it) {
        const int c = s.count(B);
        if (c >= k) {
            lo = B;
            if (c <= cap) break;
        } else {
            hi = B;
        }
        if (lo == -INFINITY) {
            B -= step;
            step *= 2.f;
        } else {
            B = 0.5f * lo + 0.5f * hi;
        }
    }
    return lo;
}

// The k best of a block's elements (nv vectors at x, then the ntail elements xt; none is NaN or +inf; the row's element e0 is the
// first) whatever their values: all elements above some t, ranked, and where they are fewer than k the first of those equal to t
// in the order of their index.  t is the maximum m where n >= k have it, -inf where up to CAND are above that, else found bit by
// bit in the order of floats, a count of the block a bit, until k to CAND are at or above it or all bits are known.  A row of
// 32,000 bf16 logits of which 10 are not masked, k = 64: 25 us; k rounds of a block-wide maximum, the next smaller key each, took
// 320; 20,000 equal rows of 1,000 fp32, k = 20: 37 and 190.  Returns how many there are.
template <typename T, int NT, int CAND, typename F>
__device__ __forceinline__ int score_select(tok_in<T> x, int nv, int ntail, float xt, int e0, int k, float m, float n,
                                            uint64_t* cand, int* ncand, int* tally, const F& emit) {
    constexpr int VEC = TokElem<T>::VEC, NW = NT / 64;
    constexpr int LOW = sizeof(T) == 4 ? 0 : __is_same(T, bf16_t) ? 16 : 13;       // bits that the type's values do not use
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // the sum of a number that each wave has; before: of the waves below this one
    const auto total = [&](int mine, int& before) {
        before = 0;
        if constexpr (NW == 1) return mine;
        __syncthreads();
        if (lane == 0) tally[wave] = mine;
        __syncthreads();
        int all = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            before += w < wave ? tally[w] : 0;
            all += tally[w];
        }
        return all;
    };
    const auto above = [&](float t) {                        // elements >= t
        int c = (int)__popcll(__ballot(tid < ntail && xt >= t)), before;
        for (int v0 = 0; v0 < nv; v0 += NT) {
            const bool in = v0 + tid < nv;
            u32x4_t r{};
            if (in) r = tok_ld16<T>(x + (int64_t)(v0 + tid) * VEC);
#pragma unroll
            for (int e = 0; e < VEC; ++e) c += (int)__popcll(__ballot(in && TokElem<T>::get(r, e) >= t));
        }
        return total(c, before);
    };
    constexpr uint32_t NONE = 0x007fffffu;                   // -inf in the order of floats
    float ge, gt;                                            // equal: >= ge and not >= gt; larger: >= gt
    int larger;
    if (n >= (float)k) {
        ge = m;
        gt = INFINITY;
        larger = 0;
    } else {
        ge = -INFINITY;
        gt = tok_unorder(NONE + 1);
        larger = above(gt);
        if (larger > CAND) {
            uint32_t t = 0;
            for (int bit = 31; bit >= LOW && larger > CAND; --bit) {
                const uint32_t c = t | 1u << bit;
                const int have = c <= NONE ? larger : above(tok_unorder(c));
                if (have >= k) {
                    t = c;
                    larger = have;
                }
            }
            ge = gt = tok_unorder(t);
            if (larger > CAND) {                             // equal ones at t: as many as there are
                gt = tok_unorder(t + (1u << LOW));
                larger = above(gt);
            }
        }
    }
    __syncthreads();
    if (tid == 0) *ncand = 0;
    __syncthreads();
    const int need = k - larger;                             // of the equal ones
    int ties = 0;
    const auto chunk = [&](const float* f, int have, int at) {
        uint32_t eq = 0;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const bool in = e < have, big = in && f[e] >= gt;
            if (in && !big && f[e] >= ge) eq |= 1u << e;
            if (larger && __ballot(big)) {
                if (big) cand[atomicAdd(ncand, 1)] = tok_key(f[e], at + e);        // up to CAND
            }
        }
        if (ties < need) {
            const int mine = __popc(eq);
            int below = 0, all = 0, before;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const uint64_t mask = __ballot((mine >> b) & 1);
                below += tok_below(mask) << b;
                all += (int)__popcll(mask) << b;
            }
            all = total(all, before);
            int rank = ties + before + below;
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if ((eq >> e) & 1) {
                    if (rank < need) emit(larger + rank, tok_key(f[e], at + e));
                    ++rank;
                }
            ties += all;
        }
    };
    float f[VEC];
    for (int v0 = 0; v0 < nv && (larger || ties < need); v0 += NT) {
        const int v = v0 + tid;
        u32x4_t r{};
        if (v < nv) r = tok_ld16<T>(x + (int64_t)v * VEC);
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] = TokElem<T>::get(r, e);
        chunk(f, v < nv ? VEC : 0, e0 + v * VEC);
    }
    f[0] = xt;
    chunk(f, tid < ntail ? 1 : 0, e0 + nv * VEC + tid);
    __syncthreads();
    tok_rank<NT>(cand, larger, k, emit);
    return need > 0 ? larger + min(ties, need) : k;
}

template <typename T, int NT, int NV>
__global__ __launch_bounds__(NT) __attribute__((amdgpu_waves_per_eu(NV == 16 ? 4 : 5))) void tok_score_kernel(ScoreArgs a) {
    constexpr int VEC = TokElem<T>::VEC, NW = NT / 64;
    // one-wave rows: 6 KB of lists a block, or LDS would keep waves away
    constexpr int SPECIAL = NT == 64 ? 192 : NT == 256 ? 128 : 64;     // vectors a wave
    constexpr int CAND = NT == 64 ? 256 : 1024;       // one wave: what it can sort
    __shared__ float red[NW][3];
    __shared__ int tally[NW];
    __shared__ TokSpecial<SPECIAL> lists[NW];
    __shared__ __attribute__((aligned(16))) uint64_t cand[CAND];
    __shared__ int ncand;                                    // over CAND: some list did not fit
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    TokSpecial<SPECIAL>& list = lists[wave];
    const int nvec_row = a.r.V / VEC;
    const int64_t u = a.r.u0 + blockIdx.x;
    const int64_t row = a.nseg == 1 ? u : u / a.nseg;
    const int seg = (int)(u - row * a.nseg);
    int64_t tgt = 0;
    if (a.y) {
        tgt = score_target(a, row);
        if (tgt == a.ignore) {
            if (a.nseg == 1) score_skip(a, row, tid, NT);
            return;
        }
    }
    tok_in<T> x = tok_row<T>(a.r, row);
    const bool valid_t = !a.y || (uint64_t)tgt < (uint64_t)a.r.V;
    float xt = 0.f;
    if (a.y && valid_t && a.nseg == 1) xt = TokElem<T>::one(x[tgt]);
    const int v0 = seg * a.segvec;
    const int nv = min(a.segvec, nvec_row - v0);
    const int ntail = seg == a.nseg - 1 ? a.r.V - nvec_row * VEC : 0;
    const int e0 = v0 * VEC;                             // the segment's first element
    x += e0;
    TokSeg<T, NT, NV> s;
    s.load(x, nv, ntail);
    const float tm = s.max_of();
    const float wm0 = tok_group<64, TokMax>(tm);
    float wb = wm0;
    if (a.k > 1) {
        // this wave's share of the bound
        if constexpr (NW > 1) wb = tok_kth_bound(tm, (a.k + NW - 1) / NW);
        else if (a.kj == 0) wb = tok_kth_bound(tm, a.k);
        else wb = tok_counted_bound(s, tm, wm0, a.k, a.kj, min(a.k + (a.k >> 1) + 16, SPECIAL));
    }
    if (lane == 0) {
        red[wave][0] = wm0;
        red[wave][1] = wb;
    }
    if (tid == 0) ncand = 0;
    __syncthreads();
    float m = red[0][0], B = red[0][1];
#pragma unroll
    for (int w = 1; w < NW; ++w) {
        m = tok_max(m, red[w][0]);
        B = fminf(B, red[w][1]);
    }
    if (a.k <= 1) B = m;
    const TokRef ref = tok_ref(m, a.r.c);
    ScoreSums sum{0.f, 0.f, 0.f};
    int chain = -1, nl = 0;                                  // the wave's vectors
    if (B > -INFINITY) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (i * NT < nv) {
                float cs = 0.f, cw = 0.f;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float d = __builtin_fmaf(TokElem<T>::get(s.r[i], e), ref.c, -ref.mc);
                    const float ev = tok_exp2(d);
                    cs += ev;
                    cw = __builtin_fmaf(ev, tok_max(d, -200.f), cw);
                }
                const bool top = s.vm[i] == m;
                list.push(s.vm[i] >= B, s.r[i], i * NT + tid, top, chain, nl);
                sum.S += top ? 0.f : cs;
                sum.W += top ? 0.f : cw;
            }
        }
        tok_wave_fence();
        for (; chain >= 0; chain = list.next[chain])
            if (list.at[chain] < 0)
                for (int e = 0; e < VEC; ++e) sum.add(list.template get<T>(chain, e), ref);
        if (tid < ntail) sum.add(s.xt, ref);
        if (nl > SPECIAL) {
            if (lane == 0) atomicAdd(&ncand, CAND + 1);
        } else if (a.k) {
            // the wave's candidates, one atomic for all that a step finds; their order does not matter
            int have = 0;
            const auto put = [&](bool hit, uint64_t key) {
                const uint64_t mask = __ballot(hit);
                if (mask == 0) return;
                int base = have;
                if constexpr (NW > 1) {
                    if (lane == 0) base = atomicAdd(&ncand, (int)__popcll(mask));
                    base = __builtin_amdgcn_readfirstlane(base);
                }
                const int at = base + tok_below(mask);
                if (hit && at < CAND) cand[at] = key;
                have += (int)__popcll(mask);
            };
            for (int b = 0; b < nl * VEC; b += 64) {
                const int i = b + lane, slot = min(i / VEC, nl - 1), e = i & (VEC - 1);
                const float xv = list.template get<T>(slot, e);
                put(i < nl * VEC && xv >= B, tok_key(xv, e0 + list.vec(slot) * VEC + e));
            }
            if (ntail && wave == 0) put(tid < ntail && s.xt >= B, tok_key(s.xt, e0 + nv * VEC + tid));
            if (NW == 1 && lane == 0) ncand = have;
        }
    }
    float S = tok_group<64, TokSum>(sum.S), W = tok_group<64, TokSum>(sum.W), n = tok_group<64, TokSum>(sum.n);
    __syncthreads();                                         // red has been read
    if (lane == 0) {
        red[wave][0] = S;
        red[wave][1] = W;
        red[wave][2] = n;
    }
    __syncthreads();                                         // the sums and the candidates are complete
    const int nc = ncand;
    const bool slow = !(B > -INFINITY) || nc > CAND;
    if (a.k == 0 && !slow && wave) return;                   // the rest is one wave's work
    if (slow) {
        // thousands of vectors at the bound (equal values), or fewer than k elements left: element by element, read again
        sum = ScoreSums{0.f, 0.f, 0.f};
        for (int v = tid; v < nv; v += NT) {
            const u32x4_t r = tok_ld16<T>(x + (int64_t)v * VEC);
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum.add(TokElem<T>::get(r, e), ref);
        }
        if (tid < ntail) sum.add(s.xt, ref);
        S = tok_group<64, TokSum>(sum.S);
        W = tok_group<64, TokSum>(sum.W);
        n = tok_group<64, TokSum>(sum.n);
        __syncthreads();
        if (lane == 0) {
            red[wave][0] = S;
            red[wave][1] = W;
            red[wave][2] = n;
        }
        __syncthreads();
    }
    S = red[0][0];
    W = red[0][1];
    n = red[0][2];
#pragma unroll
    for (int w = 1; w < NW; ++w) {
        S += red[w][0];
        W += red[w][1];
        n += red[w][2];
    }
    const float sc = tok_exp2(-ref.dmax);
    W = (W - ref.dmax * S) * sc;
    S *= sc;
    if (m == INFINITY) S = NAN;
    float lnS = 0.f;
    if (a.nseg == 1)
        lnS = score_finish(a, row, m, n, S, W, xt, valid_t, tid == 0);
    else if (tid == 0)
        a.part[u] = make_float4(m, n, S, W);
    if (a.k) {
        int done = 0;
        const auto emit = [&](int rank, uint64_t key) {
            if (a.nseg == 1) {
                a.ids[row * a.k + rank] = tok_key_index(key);
                a.top[row * a.k + rank] = score_toplp(a, tok_key_value(key), m, lnS);
            } else {
                a.keys[u * a.k + rank] = key;
            }
        };
        if (S == S) {                                        // a row (or segment) with a NaN or +inf logit has no ranking
            if (slow) {
                done = score_select<T, NT, CAND>(x, nv, ntail, s.xt, e0, a.k, m, n, cand, &ncand, tally, emit);
            } else {
                done = nc < a.k ? nc : a.k;
                tok_rank<NT>(cand, nc, a.k, emit);
            }
        }
        for (int j = done + tid; j < a.k; j += NT) {         // fewer than k elements
            if (a.nseg == 1) {
                a.ids[row * a.k + j] = -1;
                a.top[row * a.k + j] = NAN;
            } else {
                a.keys[u * a.k + j] = 0;
            }
        }
    }
}

// Joins the segments of a row.  The sums are rescaled to the row's maximum, a segment a lane, and added by a fixed tree.  Of
// the sorted lists of keys: with j = ceil(k / lists), the smallest of the j-th keys has at least k keys at or above it, and so
// has the largest of the k-th keys; what lies below both is dropped, the rest (about 1.5 k) ranked by counting.  Four waves a row
// share the keys (fp32, rows of 4 lists: 48 rows of lists of 16 4.0 us, with one wave 5.0; of 32 4.4 and 8.0; 2,000 rows of 64
// 12.0 and 16.8); one wave where the barriers would cost more: up to 32 keys (2,000 rows of lists of 8: 6.2 us, with four waves
// 8.8; 8 rows: 3.7 and 3.8), and up to 96 where the rows fill the chip (2,000 rows of lists of 16: 7.1 and 9.0).
constexpr int JOIN_CAND = 1024;
template <int NT> __global__ __launch_bounds__(NT) void tok_score_join_kernel(ScoreArgs a, int dtype) {
    __shared__ __attribute__((aligned(16))) uint64_t cand[JOIN_CAND];
    __shared__ uint64_t best[NT / 64];
    __shared__ int ncand;
    const int tid = threadIdx.x, lane = tid & 63;
    const int64_t row = a.r.u0 + blockIdx.x;
    const int nk = a.nseg * a.k;
    const uint64_t* keys = a.keys + row * nk;
    // every load that the row needs is under way before the first is waited for
    float4 p = make_float4(-INFINITY, 0.f, 0.f, 0.f);
    uint64_t first = 0, kth = 0;
    if (lane < a.nseg) {
        p = a.part[row * a.nseg + lane];
        if (a.k) {
            first = keys[lane * a.k];
            kth = keys[lane * a.k + a.k - 1];
        }
    }
    int64_t tgt = 0;
    if (a.y) tgt = score_target(a, row);
    if (a.y && tgt == a.ignore) {
        score_skip(a, row, tid, NT);
        return;
    }
    const bool valid_t = !a.y || (uint64_t)tgt < (uint64_t)a.r.V;
    float xt = 0.f;
    if (a.y && valid_t)
        xt = dtype == 0 ? tok_row<float>(a.r, row)[tgt]
             : dtype == 1 ? bf2f(tok_row<bf16_t>(a.r, row)[tgt]) : (float)tok_row<f16_t>(a.r, row)[tgt];
    if (tid == 0) ncand = 0;
    const float m = tok_group<64, TokMax>(p.x);
    float n = 0.f, S = p.z, W = 0.f;                         // a segment of nothing but -inf: 0, or NaN
    if (p.x == m) {
        n = p.y;
        W = p.w;
    } else if (p.x > -INFINITY) {
        const float d = (p.x - m) * a.r.c, f = tok_exp2(d);
        S = (p.y + p.z) * f;
        W = f > 0.f ? f * (p.w + tok_max(d, -200.f) * (p.y + p.z)) : 0.f;
    }
    n = tok_group<64, TokSum>(n);
    S = tok_group<64, TokSum>(S);
    W = tok_group<64, TokSum>(W);
    const float lnS = score_finish(a, row, m, n, S, W, xt, valid_t, tid == 0);
    if (a.k == 0) return;
    int done = 0;
    if (S == S) {                                            // a row with a NaN or +inf logit has no ranking
        // each wave works the bound out for itself
        const int live = (int)__popcll(__ballot(first != 0));
        const int j = live ? (a.k + live - 1) / live : 1;
        uint64_t B = tok_group<64, TokMin>(first ? keys[lane * a.k + j - 1] : ~(uint64_t)0);
        kth = tok_group<64, TokTop>(kth);
        if (kth > B) B = kth;
        if (B == 0) B = 1;                                   // key 0: no element
        __syncthreads();
        for (int i0 = 0; i0 < nk; i0 += NT) {
            const uint64_t key = i0 + tid < nk ? keys[i0 + tid] : 0;
            const uint64_t mask = __ballot(key >= B);
            if (mask) {
                int base = 0;
                if (lane == 0) base = atomicAdd(&ncand, (int)__popcll(mask));
                const int at = __builtin_amdgcn_readfirstlane(base) + tok_below(mask);
                if (key >= B && at < JOIN_CAND) cand[at] = key;
            }
        }
        __syncthreads();
        const int nc = ncand;
        const auto put = [&](int rank, uint64_t key) {
            a.ids[row * a.k + rank] = tok_key_index(key);
            a.top[row * a.k + rank] = score_toplp(a, tok_key_value(key), m, lnS);
        };
        if (nc <= JOIN_CAND) {
            done = nc < a.k ? nc : a.k;
            tok_rank<NT>(cand, nc, a.k, put);
        } else {                                             // lists that lie across each other: k rounds of the next largest
            uint64_t last = ~0ull;
            for (; done < a.k; ++done) {
                uint64_t bk = 0;
                for (int i = tid; i < nk; i += NT) {
                    const uint64_t key = keys[i];
                    if (key < last && key > bk) bk = key;
                }
                bk = tok_group<64, TokTop>(bk);
                if (lane == 0) best[tid >> 6] = bk;
                __syncthreads();
#pragma unroll
                for (int w = 0; w < NT / 64; ++w) bk = best[w] > bk ? best[w] : bk;
                __syncthreads();
                if (bk == 0) break;
                last = bk;
                if (tid == 0) put(done, bk);
            }
        }
    }
    for (int r = done + tid; r < a.k; r += NT) {             // fewer than k elements
        a.ids[row * a.k + r] = -1;
        a.top[row * a.k + r] = NAN;
    }
}

// Keys of a narrow row (index < 512): 16-bit types fit (order, index) in 32 bits, fp32 takes 64
template <typename T> struct NarrowKey {
    typedef uint32_t type;
    static __device__ __forceinline__ uint32_t make(float x, int i) {
        return (tok_order(x) & 0xffff0000u) | (uint32_t)(0xffff - i);
    }
    static __device__ __forceinline__ int index(uint32_t k) { return 0xffff - (int)(k & 0xffffu); }
    static __device__ __forceinline__ float value(uint32_t k) {
        return tok_unorder((k & 0xffff0000u) | ((k >> 31) ? 0u : 0xffffu));
    }
};
template <> struct NarrowKey<f16_t> {       // fp16 values need 13 more bits than bf16's: order their own 16 bits
    typedef uint32_t type;
    static __device__ __forceinline__ uint32_t make(float x, int i) {
        const uint32_t b = __builtin_bit_cast(uint16_t, (f16_t)(x + 0.0f));
        const uint32_t o = (b & 0x8000u) ? (b ^ 0xffffu) : (b | 0x8000u);
        return (o << 16) | (uint32_t)(0xffff - i);
    }
    static __device__ __forceinline__ int index(uint32_t k) { return 0xffff - (int)(k & 0xffffu); }
    static __device__ __forceinline__ float value(uint32_t k) {
        const uint32_t o = k >> 16;
        return (float)__builtin_bit_cast(f16_t, (uint16_t)((o & 0x8000u) ? (o ^ 0x8000u) : (o ^ 0xffffu)));
    }
};
template <> struct NarrowKey<float> {
    typedef uint64_t type;
    static __device__ __forceinline__ uint64_t make(float x, int i) { return tok_key(x, i); }
    static __device__ __forceinline__ int index(uint64_t k) { return tok_key_index(k); }
    static __device__ __forceinline__ float value(uint64_t k) { return tok_key_value(k); }
};
// Up to this many alternatives of a narrow row by rounds of the group's best head, more by sorting the row (120,000 rows of 40
// fp32 logits: k = 12 27 us, sorted 29; k = 20 36 and 30; k = 40 56 and 30.  Of 200: k = 20 136 and 148, k = 40 232 and 144).
// Groups of 64 lanes get no more than score_narrow_takes lets through.
template <int G> constexpr int NARROW_ROUNDS = G == 8 ? 16 : G == 16 ? 20 : 24;

template <typename T, int G>
__global__ __launch_bounds__(256) void tok_score_narrow_kernel(ScoreArgs a) {
    typedef NarrowKey<T> NK;
    typedef typename NK::type K;
    constexpr int RB = 256 / G;
    const int gl = threadIdx.x & (G - 1), gr = threadIdx.x / G;
    const int V = a.r.V;
    const int64_t r0 = (a.r.u0 + blockIdx.x) * RB;
    const int64_t row = r0 + gr;
    const bool there = row < a.r.rows;
    int64_t tgt = 0;
    if (a.y && there) tgt = score_target(a, row);
    const bool skip = a.y && tgt == a.ignore;
    const bool live = there && !skip;
    const bool valid_t = !a.y || (uint64_t)tgt < (uint64_t)V;
    tok_in<T> x = live ? tok_row<T>(a.r, row) : (tok_in<T>)0;
    float xt = 0.f;
    if (live && a.y && valid_t && gl == 0) xt = TokElem<T>::one(x[tgt]);
    float f[8];
    tok_narrow_load<T>(x, V, gl * 8, live, f);
    float m = tok_max(tok_max3(tok_max3(f[0], f[1], f[2]), f[3], f[4]), tok_max3(f[5], f[6], f[7]));
    m = tok_group<G, TokMax>(m);
    const TokRef ref = tok_ref(m, a.r.c);
    ScoreSums sum{0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 8; ++e) sum.add(f[e], ref);
    float S = tok_group<G, TokSum>(sum.S), W = tok_group<G, TokSum>(sum.W), n = tok_group<G, TokSum>(sum.n);
    const float sc = tok_exp2(-ref.dmax);
    W = (W - ref.dmax * S) * sc;
    S *= sc;
    if (m == INFINITY) S = NAN;
    float lnS = 0.f;
    if (live) lnS = score_finish(a, row, m, n, S, W, xt, valid_t, gl == 0);
    else if (there) score_skip(a, row, gl, G);
    if (a.k) {
        K h[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            // NaN and what lies behind the row are not ranked: key 0
            const bool in = gl * 8 + e < V && f[e] == f[e];
            h[e] = in ? NK::make(f[e], gl * 8 + e) : (K)0;
        }
        tok_sort_lane<8>(h);
        if (G < 64 && a.k > NARROW_ROUNDS<G>) {
            tok_sort_group<G, 8>(h, gl);
            const int at = gl * 8;
            if (live && at < a.k) {
                int64_t id[8];
                float lp[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const K key = S == S ? h[e] : (K)0;
                    id[e] = key ? NK::index(key) : -1;
                    lp[e] = key ? score_toplp(a, NK::value(key), m, lnS) : NAN;
                }
                tok_out<int64_t> ids = (tok_out<int64_t>)a.ids + row * a.k + at;
                tok_out<float> top = (tok_out<float>)a.top + row * a.k + at;
                if (at + 8 <= a.k) {
#pragma unroll
                    for (int e = 0; e < 8; e += 2)
                        tok_st16<int64_t>(ids + e, u32x4_t{(uint32_t)id[e], (uint32_t)(id[e] >> 32), (uint32_t)id[e + 1],
                                                           (uint32_t)(id[e + 1] >> 32)});
#pragma unroll
                    for (int e = 0; e < 8; e += 4) tok_st16<float>(top + e, TokElem<float>::pack(lp + e));
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (at + e < a.k) {
                            ids[e] = id[e];
                            top[e] = lp[e];
                        }
                }
            }
            return;
        }
        K keep = 0;
        for (int j = 0; j < a.k; ++j) {
            const K top = tok_group<G, TokTop>(h[0]);
            if (top == h[0]) {                           // keys differ, so one lane's head goes (or all are 0)
#pragma unroll
                for (int e = 0; e < 7; ++e) h[e] = h[e + 1];
                h[7] = 0;
            }
            if ((j & (G - 1)) == gl) keep = S == S ? top : (K)0;
            if ((j & (G - 1)) == G - 1 || j == a.k - 1) {
                const int at = (j & ~(G - 1)) + gl;      // G results at a time, one a lane
                if (live && at <= j) {
                    a.ids[row * a.k + at] = keep ? NK::index(keep) : -1;
                    a.top[row * a.k + at] = keep ? score_toplp(a, NK::value(keep), m, lnS) : NAN;
                }
            }
        }
    }
}

// Many short rows: a row a lane.  The row's eighths keep their maxima in registers; a round takes the lowest one that holds the
// maximum, reads those 8 elements of the row in LDS, and marks the lowest that holds it as taken (NaN, which no maximum and no
// comparison sees).  ~65 operations a round; a pass over the row's registers takes ~180.  The alternatives go out through
// LDS too.
template <typename T> __global__ __launch_bounds__(64) void tok_score_lane_kernel(ScoreArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint64_t lane_lds[];
    T* rows = reinterpret_cast<T*>(lane_lds);
    const int V = a.r.V, k = a.k, lane = threadIdx.x;
    const int64_t row0 = (a.r.u0 + blockIdx.x) * 64, row = row0 + lane;
    const int nrow = a.r.rows - row0 < 64 ? (int)(a.r.rows - row0) : 64;
    const bool there = lane < nrow;
    int64_t tgt = 0;
    if (a.y && there) tgt = score_target(a, row);
    tok_stage_rows<T>(a.r, row0, nrow, rows);
    const bool skip = a.y && tgt == a.ignore, valid_t = !a.y || (uint64_t)tgt < (uint64_t)V;
    const T* x = rows + lane * V;                            // lanes behind the last row read what is there, and write nothing
    float xt = 0.f;
    if (a.y && valid_t && !skip) xt = TokElem<T>::one(x[tgt]);
    TokLane<T> l;
    l.load(x, V, -INFINITY);
    const float m = l.max_of(V, -INFINITY);
    const TokRef ref = tok_ref(m, a.r.c);
    ScoreSums sum{0.f, 0.f, 0.f};
    l.each(V, [&](int, float f) { sum.add(f, ref); });
    const float sc = tok_exp2(-ref.dmax);
    const float W = (sum.W - ref.dmax * sum.S) * sc, S = m == INFINITY ? NAN : sum.S * sc;
    float lnS = 0.f;
    if (there && !skip) lnS = score_finish(a, row, m, sum.n, S, W, xt, valid_t, true);
    else if (there) score_skip(a, row, 0, 0);
    if (k) {
        T* mine = rows + lane * V;
        int* ids = reinterpret_cast<int*>(reinterpret_cast<char*>(lane_lds) + (64 * V * sizeof(T) + 15) / 16 * 16);
        float* lps = reinterpret_cast<float*>(ids + 64 * k);
        float cm[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            cm[i] = NAN;
            if (i * 8 < V) {                                 // pads are -inf: an eighth of nothing else has maximum -inf
#pragma unroll
                for (int e = 0; e < 8; e += 2) cm[i] = tok_max3(cm[i], l.f[i * 8 + e], l.f[i * 8 + e + 1]);
            }
        }
        for (int j = 0; j < k; ++j) {
            float top = NAN;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i * 8 < V) top = tok_max(top, cm[i]);
            int c = 0;
#pragma unroll
            for (int i = 7; i >= 0; --i)
                if (i * 8 < V) c = cm[i] == top ? i : c;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = c * 8 + e < V ? TokElem<T>::one(mine[c * 8 + e]) : NAN;
            int at = -1;
#pragma unroll
            for (int e = 7; e >= 0; --e) at = v[e] == top ? e : at;
            float rest = NAN;
#pragma unroll
            for (int e = 0; e < 8; ++e) rest = tok_max(rest, e == at ? NAN : v[e]);
            if (at >= 0) mine[c * 8 + at] = TokElem<T>::put(NAN);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i * 8 < V) cm[i] = i == c ? rest : cm[i];
            int id = at < 0 || !(S == S) ? -1 : c * 8 + at;  // a row with a NaN or +inf logit has no ranking
            float lp = id < 0 ? NAN : score_toplp(a, top, m, lnS);
            if (skip) {
                id = -1;
                lp = -INFINITY;
            }
            ids[lane * k + j] = id;
            lps[lane * k + j] = lp;
        }
        tok_wave_fence();
        for (int i = lane; i < nrow * k; i += 64) {
            a.ids[row0 * k + i] = ids[i];
            a.top[row0 * k + i] = lps[i];
        }
    }
}

// ---- backward ----------------------------------------------------------------------------------------------------------
struct ScoreGradArgs {
    TokRows r;
    int64_t y, t0, t1, ignore;
    int y64, chunks;
    const float *glp, *gent, *stat;  // glp / gent: 0 = no such gradient
    int64_t dx;                      // [rows][V]
};
// dx = ( gl [v = target] - q (gl + gh (ln q + H)) ) / T,  log2 q = fma(x - m, c, -l2S)
struct ScoreCoef {
    float m, l2S, a, b, gl;          // -q (a + b log2 q) + [target] gl
};
__device__ __forceinline__ ScoreCoef score_coef(const ScoreGradArgs& a, int64_t row, bool valid_t) {
    const float* st = a.stat + row * 3;
    float gl = a.glp ? a.glp[row] : 0.f;
    const float gh = a.gent ? a.gent[row] : 0.f;
    if (!valid_t && a.glp) gl = NAN;                         // a target outside the vocabulary: loud
    ScoreCoef k;
    k.m = st[0];
    k.l2S = st[1];
    k.gl = gl * a.r.inv_t;
    k.a = (gl + gh * st[2]) * a.r.inv_t;
    k.b = gh * 0.6931471805599453f * a.r.inv_t;
    if (k.l2S == INFINITY) k.a = k.b = k.gl = 0.f;            // an empty row has no gradient
    return k;
}
__device__ __forceinline__ float score_dx(const ScoreCoef& k, float c, float x) {
    const float l = __builtin_fmaf(x - k.m, c, -k.l2S);      // log2 q
    return -tok_exp2(l) * __builtin_fmaf(k.b, tok_max(l, -200.f), k.a);
}

// a thread owns U vectors, 256 apart: one read and one write an element, ~11 operations; HBM-bound
template <typename T>
__global__ __launch_bounds__(256) void tok_score_grad_kernel(ScoreGradArgs a) {
    constexpr int VEC = TokElem<T>::VEC, U = 4;
    const int tid = threadIdx.x;
    const int nvec = a.r.V / VEC, ntail = a.r.V - nvec * VEC;
    const int64_t u = a.r.u0 + blockIdx.x;
    const int64_t row = u / a.chunks;
    const int ch = (int)(u - row * a.chunks);
    const int64_t i0 = a.r.n1 == a.r.rows ? 0 : (int64_t)((uint32_t)row / (uint32_t)a.r.n1);
    const int64_t tgt = a.y ? tok_int(a.y, a.y64, i0 * a.t0 + (row - i0 * a.r.n1) * a.t1) : 0;
    const bool skip = a.y && tgt == a.ignore, valid_t = !a.y || (uint64_t)tgt < (uint64_t)a.r.V;
    tok_out<T> o = (tok_out<T>)a.dx + row * a.r.V;
    tok_in<T> x = tok_row<T>(a.r, row);
    const int b0 = ch * 256 * U;
    ScoreCoef k{};
    if (!skip) k = score_coef(a, row, valid_t);
    const int tv = a.y ? (int)tgt / VEC : -1, te = a.y ? (int)tgt - tv * VEC : 0;
    u32x4_t r[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int v = b0 + i * 256 + tid;
        if (!skip && v < nvec) r[i] = tok_ld16<T>(x + (int64_t)v * VEC);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int v = b0 + i * 256 + tid;
        if (v < nvec) {
            float f[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) f[e] = skip ? 0.f : score_dx(k, a.r.c, TokElem<T>::get(r[i], e));
            if (!skip && v == tv)
#pragma unroll
                for (int e = 0; e < VEC; ++e) f[e] += e == te ? k.gl : 0.f;
            tok_st16<T>(o + (int64_t)v * VEC, TokElem<T>::pack(f));
        }
    }
    if (ch == a.chunks - 1 && tid < ntail) {
        const int e = nvec * VEC + tid;
        float f = 0.f;
        if (!skip) f = score_dx(k, a.r.c, TokElem<T>::one(x[e])) + (a.y && e == (int)tgt ? k.gl : 0.f);
        o[e] = TokElem<T>::put(f);
    }
}

template <typename T, int G>
__global__ __launch_bounds__(256) void tok_score_grad_narrow_kernel(ScoreGradArgs a) {
    constexpr int RB = 256 / G;
    const int gl = threadIdx.x & (G - 1), gr = threadIdx.x / G;
    const int V = a.r.V;
    const int64_t r0 = (a.r.u0 + blockIdx.x) * RB;
    const int64_t row = r0 + gr;
    if (row >= a.r.rows) return;
    const int64_t i0 = a.r.n1 == a.r.rows ? 0 : (int64_t)((uint32_t)row / (uint32_t)a.r.n1);
    const int64_t tgt = a.y ? tok_int(a.y, a.y64, i0 * a.t0 + (row - i0 * a.r.n1) * a.t1) : 0;
    const bool skip = a.y && tgt == a.ignore, valid_t = !a.y || (uint64_t)tgt < (uint64_t)V;
    if (gl * 8 >= V) return;
    float f[8];
    tok_narrow_load<T>(tok_row<T>(a.r, row), V, gl * 8, !skip, f);
    if (skip) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = 0.f;
    } else {
        const ScoreCoef k = score_coef(a, row, valid_t);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            f[e] = score_dx(k, a.r.c, f[e]);
            if (a.y && gl * 8 + e == (int)tgt) f[e] += k.gl;
        }
    }
    tok_narrow_store<T>((tok_out<T>)a.dx + row * V, V, gl * 8, f);
}

// ---- launchers ---------------------------------------------------------------------------------------------------------
// whole up to 8192 vectors (512 threads x 16): 2,000 rows of 32,000 fp32 logits 40 us, in two pieces 42; one row 5.4 and 8.7
static TokPlan score_plan(int64_t V, int dtype) { return tok_plan(V, tok_esize(dtype), 8192); }

// Up to this many alternatives of a row on one wave by the lanes' maxima, more by a counted bound (120,000 rows of 1,000 fp32
// logits, before the candidates were sorted: k = 20 182 us, counted 198; k = 32 250 and 247; k = 64 1,390 and 337; k = 100 4,540
// and 482)
constexpr int ONE_WAVE_LANES = 24;

// Rows of 257 to 512 elements with alternatives: a row a wave by the long rows' kernel where listing candidates costs less than
// rounds over 64 lanes (120,000 rows of 500: fp32 with k = 1 104 us, narrow 108, k = 20 139 and 300; bf16 with k = 8 136 and
// 120, k = 20 152 and 169)
static bool score_narrow_takes(int64_t V, int dtype, int k) {
    return V <= 256 || (V <= TOK_NARROW_V && k <= (dtype == 0 ? 0 : 12));
}

// segments a row is cut into (the workspace holds 16 + 8 k bytes for each when more than one)
int64_t tok_score_segments(int64_t V, int dtype) {
    return V <= TOK_NARROW_V ? 1 : score_plan(V, dtype).nseg;
}

template <typename T> static void score_wide(const ScoreArgs& a, const TokPlan& p, hipStream_t s) {
    const int64_t units = a.r.rows * p.nseg;
    const int nt = p.nt;
    if (p.nt == 64 && p.nv == 2) tok_launch(tok_score_kernel<T, 64, 2>, units, nt, 0, s, a);
    else if (p.nt == 64 && p.nv == 4) tok_launch(tok_score_kernel<T, 64, 4>, units, nt, 0, s, a);
    else if (p.nt == 64) tok_launch(tok_score_kernel<T, 64, 8>, units, nt, 0, s, a);
    else if (p.nv == 4) tok_launch(tok_score_kernel<T, 256, 4>, units, nt, 0, s, a);
    else if (p.nv == 8) tok_launch(tok_score_kernel<T, 256, 8>, units, nt, 0, s, a);
    else if (p.nt == 256) tok_launch(tok_score_kernel<T, 256, 16>, units, nt, 0, s, a);
    else tok_launch(tok_score_kernel<T, 512, 16>, units, nt, 0, s, a);
}
template <typename T> static void score_narrow(const ScoreArgs& a, hipStream_t s) {
    if (tok_lane_rows(a.r.V, sizeof(T), a.r.rows) && a.k <= 8) {        // more alternatives: rounds on 8 lanes cost less
        const size_t lds = (64 * a.r.V * sizeof(T) + 15) / 16 * 16 + 64 * a.k * 8;
        tok_launch(tok_score_lane_kernel<T>, (a.r.rows + 63) / 64, 64, lds, s, a);
        return;
    }
    const int G = tok_narrow_lanes(a.r.V);
    const int64_t rb = 256 / G;
    const int64_t units = (a.r.rows + rb - 1) / rb;
    const int nt = 256;
    if (G == 8) tok_launch(tok_score_narrow_kernel<T, 8>, units, nt, 0, s, a);
    else if (G == 16) tok_launch(tok_score_narrow_kernel<T, 16>, units, nt, 0, s, a);
    else if (G == 32) tok_launch(tok_score_narrow_kernel<T, 32>, units, nt, 0, s, a);
    else tok_launch(tok_score_narrow_kernel<T, 64>, units, nt, 0, s, a);
}

template <typename T> static void score_grad_narrow(const ScoreGradArgs& a, hipStream_t s) {
    const int G = tok_narrow_lanes(a.r.V);
    const int64_t rb = 256 / G;
    const int64_t units = (a.r.rows + rb - 1) / rb;
    const int nt = 256;
    if (G == 8) tok_launch(tok_score_grad_narrow_kernel<T, 8>, units, nt, 0, s, a);
    else if (G == 16) tok_launch(tok_score_grad_narrow_kernel<T, 16>, units, nt, 0, s, a);
    else if (G == 32) tok_launch(tok_score_grad_narrow_kernel<T, 32>, units, nt, 0, s, a);
    else tok_launch(tok_score_grad_narrow_kernel<T, 64>, units, nt, 0, s, a);
}

// dtype: 0 fp32, 1 bf16, 2 fp16.  y = 0: no targets (lp is not written).  ws: rows * segments * (16 + 8 k) bytes, 16-aligned.
void launch_tok_score(uint64_t x, int dtype, int64_t rows, int64_t n1, int64_t s0, int64_t s1, int64_t V, double temperature,
                      uint64_t y, int y64, int64_t t0, int64_t t1, int64_t ignore, int k, uint64_t lp, uint64_t ent,
                      uint64_t ids, uint64_t top, uint64_t stat, uint64_t ws, uint64_t stream) {
    if (rows <= 0) return;
    if (dtype < 0 || dtype > 2) throw std::runtime_error("token operators: unknown logits type");
    if (k < 0 || k > TOK_MAX_K || k > V) throw std::runtime_error("tok_score: top_k out of range");
    if (!ent || (lp && !y) || (k && (!ids || !top))) throw std::runtime_error("tok_score: a tensor has no storage");
    ScoreArgs a{};
    a.r = tok_rows_of(x, rows, n1, s0, s1, V, temperature);
    a.y = (int64_t)y;
    a.y64 = y64;
    a.t0 = t0;
    a.t1 = t1;
    a.ignore = ignore;
    a.k = k;
    a.lp = as_ptr<float>(y ? lp : 0);
    a.ent = as_ptr<float>(ent);
    a.ids = as_ptr<int64_t>(ids);
    a.top = as_ptr<float>(top);
    a.stat = as_ptr<float>(stat);
    a.nseg = 1;
    const hipStream_t s = as_stream(stream);
    if (score_narrow_takes(V, dtype, k)) {
        if (dtype == 0) score_narrow<float>(a, s);
        else if (dtype == 1) score_narrow<bf16_t>(a, s);
        else score_narrow<f16_t>(a, s);
        return;
    }
    const TokPlan p = score_plan(V, dtype);
    a.nseg = p.nseg;
    a.segvec = p.segvec;
    if (p.nt == 64 && k > ONE_WAVE_LANES) {
        const int64_t nvec = V / (16 / tok_esize(dtype)), lanes = nvec < 64 ? nvec : 64;
        const double q = 1.25 * k / V, n = (double)V / lanes;
        a.kj = q < 1 ? (int)ceil(lanes * (1 - pow(1 - q, n))) : (int)lanes;
    }
    if (p.nseg > 1) {
        if (!ws) throw std::runtime_error("tok_score: this shape needs a workspace");
        a.part = as_ptr<float4>(ws);
        a.keys = as_ptr<uint64_t>(ws + (uint64_t)rows * p.nseg * 16);
    }
    if (dtype == 0) score_wide<float>(a, p, s);
    else if (dtype == 1) score_wide<bf16_t>(a, p, s);
    else score_wide<f16_t>(a, p, s);
    if (p.nseg > 1) {
        const int nk = p.nseg * k;
        if (nk <= 32 || (nk <= 96 && rows > 1024)) tok_launch(tok_score_join_kernel<64>, rows, 64, 0, s, a, dtype);
        else tok_launch(tok_score_join_kernel<256>, rows, 256, 0, s, a, dtype);
    }
}

void launch_tok_score_grad(uint64_t x, int dtype, int64_t rows, int64_t n1, int64_t s0, int64_t s1, int64_t V,
                           double temperature, uint64_t y, int y64, int64_t t0, int64_t t1, int64_t ignore, uint64_t glp,
                           uint64_t gent, uint64_t stat, uint64_t dx, uint64_t stream) {
    if (rows <= 0) return;
    if (dtype < 0 || dtype > 2) throw std::runtime_error("token operators: unknown logits type");
    if (!stat || !dx) throw std::runtime_error("tok_score: a tensor has no storage");
    ScoreGradArgs a{};
    a.r = tok_rows_of(x, rows, n1, s0, s1, V, temperature);
    a.y = (int64_t)y;
    a.y64 = y64;
    a.t0 = t0;
    a.t1 = t1;
    a.ignore = ignore;
    a.glp = as_ptr<const float>(y ? glp : 0);
    a.gent = as_ptr<const float>(gent);
    a.stat = as_ptr<const float>(stat);
    a.dx = (int64_t)dx;
    const hipStream_t s = as_stream(stream);
    if (V <= TOK_NARROW_V) {
        if (dtype == 0) score_grad_narrow<float>(a, s);
        else if (dtype == 1) score_grad_narrow<bf16_t>(a, s);
        else score_grad_narrow<f16_t>(a, s);
    } else {
        const int64_t nvec = V / (16 / tok_esize(dtype));
        a.chunks = (int)((nvec + 1023) / 1024);
        const int64_t units = rows * a.chunks;
        const int nt = 256;
        if (dtype == 0) tok_launch(tok_score_grad_kernel<float>, units, nt, 0, s, a);
        else if (dtype == 1) tok_launch(tok_score_grad_kernel<bf16_t>, units, nt, 0, s, a);
        else tok_launch(tok_score_grad_kernel<f16_t>, units, nt, 0, s, a);
    }
}
