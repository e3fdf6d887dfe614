// Distillation from a teacher's top tokens: the loss of a row of student logits x and its gradient.
//
// The teacher gives K pairs (id i_k, log-probability t_k) a row; pairs whose id is outside [0, V) are absent, pairs of the
// same id add up.  With z = x / T, q = softmax(z):
//   drop  : p_k = exp(t_k) / sum_k exp(t_k)                                   loss = w T^2 sum_k p_k (ln p_k - ln q_ik)
//   bucket: p_k = exp(t_k), p_0 = max(0, 1 - sum p_k), q_0 = sum_{v not listed} q_v,
//           loss = w T^2 ( sum_k p_k (ln p_k - ln q_ik) + p_0 (ln p_0 - ln q_0) )       (no bucket where ln q_0 < -745)
//   gradient, with P = sum p_k, A = P + p_0 (drop: A = P):
//           dx_v = w T ( A q_v - p_v ) for listed v,   w T (A q_0 - p_0) (q_v / q_0) for the others (drop: w T P q_v)
// A row of weight 0 is not read: loss and gradient 0.
//
// A student may be so sure of its list that q_0 is nothing in fp32 (88 T below the row's maximum), and that is where the bucket
// has most to say.  So q_0 has a reference of its own, mu: the row's maximum m while the sum relative to it is 2^-64 or more (what
// underflows then, 2^-126 an element, does not count), else the largest unlisted element, in a second look that only such rows
// take.  ln q_0 = (mu - m) / T + ln rest - ln sum, and q_v / q_0 = exp((x_v - mu) / T) / rest.  Below exp(-745), where 64 bits end,
// the rest counts as ruled out (a finite mask value), as -inf does.
//
// The loss of a good student is a small difference of large terms (its digits go with the rounding of ln sum alone), so a
// row's sums are fp32 but its logarithms and K terms fp64: K + 3 transcendentals a row, next to V fp32 ones.
//
// One pass (tok_distill_kernel, GRAD): a block holds the row in registers, so the gradient needs no second read of HBM:
// 2 V elements moved a row, which is the floor.  Listed tokens are marked in an LDS bitmap (one byte a 16-bit vector), so
// q_0 is summed over the others directly and not as 1 - sum.  Rows too long for a block's registers, and the autograd
// form, whose gradient comes later, take the statistics first (joined over segments where a row is cut) and the gradient in
// a second launch.
#include "token.h"

constexpr int DIST_MAX_K = 256;

struct DistArgs {
    TokRows r;
    int64_t ids;
    const float *t, *w;
    int id64, K, bucket;
    int nseg, segvec;
    float T;
    float* loss;
    int64_t dx;           // [rows][V], one-pass form
    float4* stat;         // for the gradient launch, two a row: (m, l2S, A, -) and (mu, l2u, B, -) of DistRow
    float* pk;            // [rows][K]: p of the entry's token
    float4* part;         // nseg > 1: (mu, n, S, m) of each segment: its sums relative to mu (bucket: of the unlisted), its maximum
};

// The K entries of a row in LDS: id (-1: absent), the student's logit there, p
struct DistEntries {
    int id[DIST_MAX_K];
    float x[DIST_MAX_K], t[DIST_MAX_K], p[DIST_MAX_K];
};
struct DistRow {
    float m, l2S, A;      // listed: A q - p, log2 q = (x - m) c - l2S
    float mu, l2u, B;     // others: B exp2((x - mu) c - l2u)
};
constexpr float DIST_FAR = 0x1p-64f;      // a rest below this, relative to the row's maximum, takes a reference of its own

__device__ __forceinline__ double group_sum64(double v) { return tok_group<64, TokSum>(v); }

// Sums over a row's entries: with s = the largest t (drop mode) or 0 (bucket), e_k = exp(t_k - s),
//   tot = sum e_k,   acc = sum e_k ( (t_k - s) - (x_k - m) / T )
// one fp64 exponential an entry; p_k = e_k / tot (drop) or e_k (bucket).  An id that occurs several times is one token: each of its
// entries then also brings e_k ln( sum of the e_i of that id / e_k ) (dist_parts).
struct DistTeach {
    double tot, acc;
    __device__ __forceinline__ void add(float t, float s, float x, float m, double inv_t) {
        const double l = (double)t - (double)s, e = exp(l);
        tot += e;
        if (e != 0.0) acc += e * (l - (x == -INFINITY ? -(double)INFINITY : ((double)x - (double)m) * inv_t));
    }
};
// An entry's e ln( sum of its id's e_i / e ).  same(i): entry i has that id; t_at(i): its value.  A term of its own and in fp32: it
// is rare, and inside the fp64 loop it costs every row registers.  It may be off by some 2^-21 of e, less than ln sum is.
template <typename S, typename V>
__device__ __forceinline__ float dist_parts(int K, float t, float s, const S& same, const V& t_at) {
    float top = t, sum = 0.f;
    for (int i = 0; i < K; ++i)
        if (same(i)) top = tok_max(top, t_at(i));
    for (int i = 0; i < K; ++i)
        if (same(i)) sum += tok_exp2((t_at(i) - top) * 1.4426950408889634f);
    const float e = tok_exp2((t - s) * 1.4426950408889634f);
    return e == 0.f ? 0.f : e * (top - t + __builtin_amdgcn_logf(sum) * 0.6931471805599453f);
}
// A row's loss and the gradient's factors.  rest: the student's sum over the elements outside the list relative to mu (mu = m where
// there is nothing), listed: inside it, relative to m (drop mode: their sum counts, mu = m).  shift: ln p_k = t_k - shift.
struct DistDone {
    DistRow d;
    double kl, shift;
    bool none;
};
__device__ __forceinline__ DistDone dist_finish(const DistArgs& a, float m, float mu, double rest, double listed, double tot,
                                                double acc, float s) {
    DistDone r;
    double far = 0.0, rm = rest;                             // (mu - m) / T, the rest relative to m
    if (__builtin_expect(__ballot(mu != m) != 0, 0)) {
        far = mu == m ? 0.0 : ((double)mu - (double)m) * a.r.dinv_t;
        rm = rest * exp(far);
    }
    double sum = rm + listed;
    if (m == INFINITY) sum = (double)NAN;
    r.none = sum == 0.0;                                     // nothing left of the student: infinite loss, no gradient
    const double lnS = r.none ? 0.0 : log(sum);
    r.d.m = r.d.mu = r.none ? 0.f : m;
    r.d.l2S = r.d.l2u = r.none ? INFINITY : (float)(lnS * 1.4426950408889634);
    if (a.bucket) {
        r.shift = 0.0;
        r.kl = acc + (tot != 0.0 ? tot * lnS : 0.0);
        r.d.A = r.d.B = (float)tot;
        const double p0 = 1.0 - tot;
        const double lq0 = sum != sum ? sum : rest == 0.0 ? -(double)INFINITY
                           : listed < rm ? log1p(-listed / sum) : far + log(rest / sum);
        if (p0 > 0.0 && !(lq0 < -745.0)) {
            r.kl += p0 * (log(p0) - lq0);
            r.d.A = (float)(tot + p0);
            r.d.B = (float)((tot + p0) * (rm / sum) - p0);
            r.d.mu = mu;
            r.d.l2u = log2f((float)rest);
        }
    } else {
        const double lt = tot == 0.0 ? 0.0 : log(tot);
        r.shift = (tot == 0.0 ? 0.0 : (double)s) + lt;
        r.kl = tot == 0.0 ? 0.0 : acc / tot - lt + lnS;
        r.d.A = r.d.B = (float)(tot == 0.0 ? 0.0 : 1.0 + (tot - tot));        // NaN stays NaN
    }
    return r;
}
__device__ __forceinline__ float dist_q(const DistRow& d, float c, float x) {
    return tok_exp2(__builtin_fmaf(x - d.m, c, -d.l2S));
}
// an element outside the list, B still to be multiplied
__device__ __forceinline__ float dist_u(const DistRow& d, float c, float x) {
    return tok_exp2(__builtin_fmaf(x - d.mu, c, -d.l2u));
}
__device__ __forceinline__ void dist_keep(float4* stat, int64_t row, const DistRow& d) {
    stat[2 * row] = make_float4(d.m, d.l2S, d.A, 0.f);
    stat[2 * row + 1] = make_float4(d.mu, d.l2u, d.B, 0.f);
}
__device__ __forceinline__ DistRow dist_kept(const float4* stat, int64_t row) {
    const float4 l = stat[2 * row], u = stat[2 * row + 1];
    return DistRow{l.x, l.y, l.z, u.x, u.y, u.z};
}
// a listed element's A q - p; nothing where the student has nothing left
__device__ __forceinline__ float dist_l(const DistRow& d, float c, float x, float p) {
    return d.l2S == INFINITY ? 0.f : __builtin_fmaf(d.A, dist_q(d, c, x), -p);
}
// an entry's p for the gradient, in fp32
__device__ __forceinline__ float dist_p(float t, double shift) {
    return tok_exp2((float)(((double)t - shift) * 1.4426950408889634));
}

// The first wave's work on a row: the loss, and each entry's p.  n, S: the student's sums relative to mu over all elements, or
// in bucket mode over the unlisted ones.  dup: some id may occur twice; each occurrence has the whole p then.
__device__ __forceinline__ DistRow dist_epilogue(const DistArgs& a, DistEntries& E, int64_t row, float w, float m,
                                                 float mu, float n, float S, bool dup, int lane) {
    const int K = a.K;
    float s = -INFINITY;
    if (!a.bucket) {
        for (int j = lane; j < K; j += 64)
            if (E.id[j] >= 0) s = tok_max(s, E.t[j]);
        s = tok_group<64, TokMax>(s);
    }
    if (!(s > -INFINITY)) s = 0.f;
    DistTeach te{0.0, 0.0};
    for (int j = lane; j < K; j += 64)
        if (E.id[j] >= 0) te.add(E.t[j], s, E.x[j], m, a.r.dinv_t);
    te.tot = group_sum64(te.tot);
    te.acc = group_sum64(te.acc);
    bool first[DIST_MAX_K / 64], twice = false;
    float nl = 0.f, Sl = 0.f;
#pragma unroll
    for (int q = 0; q < DIST_MAX_K / 64; ++q) {
        const int j = q * 64 + lane;
        first[q] = j < K && E.id[j] >= 0;
        if (dup && first[q])
            for (int i = 0; i < j; ++i) first[q] &= E.id[i] != E.id[j];
        twice |= j < K && E.id[j] >= 0 && !first[q];
        if (a.bucket && first[q]) {
            if (E.x[j] == m) nl += m > -INFINITY ? 1.f : 0.f;
            else if (m > -INFINITY) Sl += tok_exp2((E.x[j] - m) * a.r.c);
        }
    }
    nl = tok_group<64, TokSum>(nl);
    Sl = tok_group<64, TokSum>(Sl);
    dup = __ballot(twice) != 0;
    if (__builtin_expect(dup, 0)) {
        float more = 0.f;
        for (int j = lane; j < K; j += 64)
            if (E.id[j] >= 0)
                more += dist_parts(K, E.t[j], s, [&](int i) { return E.id[i] == E.id[j]; }, [&](int i) { return E.t[i]; });
        te.acc += (double)tok_group<64, TokSum>(more);
    }
    const DistDone r = dist_finish(a, m, mu, (double)n + (double)S, (double)nl + (double)Sl, te.tot, te.acc, s);
    for (int j = lane; j < K; j += 64) E.p[j] = dist_p(E.t[j], r.shift);
    if (__builtin_expect(dup, 0)) {
        tok_wave_fence();
        float sum[DIST_MAX_K / 64];
#pragma unroll
        for (int q = 0; q < DIST_MAX_K / 64; ++q) {
            const int j = q * 64 + lane;
            sum[q] = 0.f;
            if (j < K)
                for (int i = 0; i < K; ++i) sum[q] += E.id[i] == E.id[j] ? E.p[i] : 0.f;
        }
        tok_wave_fence();
#pragma unroll
        for (int q = 0; q < DIST_MAX_K / 64; ++q)
            if (q * 64 + lane < K) E.p[q * 64 + lane] = sum[q];
    }
    if (a.pk)
        for (int j = lane; j < K; j += 64) a.pk[row * K + j] = E.p[j];
    if (lane == 0) {
        a.loss[row] = (float)((double)w * (double)a.T * (double)a.T * r.kl);
        if (a.stat) dist_keep(a.stat, row, r.d);
    }
    return r.d;
}

template <typename T> __device__ __forceinline__ void dist_load_entry(const DistArgs& a, DistEntries& E, int64_t row, tok_in<T> x,
                                                                      int j) {
    int64_t id = tok_int(a.ids, a.id64, row * a.K + j);
    const bool in = (uint64_t)id < (uint64_t)a.r.V;
    E.id[j] = in ? (int)id : -1;
    E.t[j] = a.t[row * a.K + j];
    E.x[j] = in ? TokElem<T>::one(x[id]) : 0.f;
}
// One element's share of the sums; skip: listed, in bucket mode
struct DistSums {
    float S, n;
    __device__ __forceinline__ void add(float x, const TokRef& ref, bool skip) {
        const bool is = x == ref.meq;
        S += is || skip ? 0.f : tok_exp2(__builtin_fmaf(x, ref.c, -ref.mc));
        n += is && !skip ? 1.f : 0.f;
    }
};

// f(element) over a thread's elements of a segment that no bit marks, read again.  Element by element in a loop: unrolled, its
// masks would take the scalar registers of a wave from the kernel that this is the rare part of (8,192 x 8,000 bf16, K = 64, tail
// bucket: 69 us, 65).  It is worth a second read: 8,192 x 32,000 bf16 with every row sure of its list 433 us, 224 else.
template <typename T, int NT, typename F>
__device__ __forceinline__ void dist_unlisted(tok_in<T> x, int nv, const uint32_t* bits, const F& f) {
    constexpr int VEC = TokElem<T>::VEC;
    for (int v = threadIdx.x; v < nv; v += NT) {
        u32x4_t r = tok_ld16<T>(x + (int64_t)v * VEC);
        uint32_t listed = bits[(v * VEC) >> 5] >> ((v * VEC) & 31);                  // a vector's bits lie in one word
#pragma unroll 1
        for (int e = 0; e < VEC; ++e, listed >>= 1) {
            if (!(listed & 1)) f(TokElem<T>::get(r, 0));
            if constexpr (VEC == 4) r = u32x4_t{r[1], r[2], r[3], 0};
            else r = u32x4_t{r[0] >> 16 | r[1] << 16, r[1] >> 16 | r[2] << 16, r[2] >> 16 | r[3] << 16, r[3] >> 16};
        }
    }
}

template <typename T, int NT, int NV, bool GRAD>
__global__ __launch_bounds__(NT) __attribute__((amdgpu_waves_per_eu(4))) void tok_distill_kernel(DistArgs a) {
    constexpr int VEC = TokElem<T>::VEC, NW = NT / 64;
    constexpr int WORDS = NT * NV * VEC / 32 + 1;
    __shared__ DistEntries E;
    __shared__ uint32_t bits[WORDS];                         // listed tokens of the segment
    constexpr int SPECIAL = NT == 64 ? 192 : NT == 256 ? 128 : NT == 512 ? 96 : 48;     // a wave
    __shared__ TokSpecial<SPECIAL> lists[NW];
    __shared__ float red[NW][3];
    __shared__ int dup, over;                                // an id occurs twice; some wave's list did not fit
    __shared__ DistRow rowd;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    TokSpecial<SPECIAL>& list = lists[wave];
    const int nvec_row = a.r.V / VEC, ntail_row = a.r.V - nvec_row * VEC;
    const int64_t u = a.r.u0 + blockIdx.x;
    const int64_t row = a.nseg == 1 ? u : u / a.nseg;
    const int seg = (int)(u - row * a.nseg);
    const float w = a.w ? a.w[row] : 1.f;
    tok_out<T> o = (tok_out<T>)a.dx + row * a.r.V;
    if (w == 0.f) {
        if (a.nseg == 1 && tid == 0) a.loss[row] = 0.f;
        if constexpr (GRAD) {
            for (int v = tid; v < nvec_row; v += NT) tok_st16<T>(o + (int64_t)v * VEC, u32x4_t{0, 0, 0, 0});
            if (tid < ntail_row) o[nvec_row * VEC + tid] = TokElem<T>::put(0.f);
        }
        return;
    }
    tok_in<T> x = tok_row<T>(a.r, row);
    const int v0 = seg * a.segvec;
    const int nv = min(a.segvec, nvec_row - v0);
    const int ntail = seg == a.nseg - 1 ? ntail_row : 0;
    const int e0 = v0 * VEC, len = nv * VEC + ntail;
    TokSeg<T, NT, NV> s;
    s.load(x + e0, nv, ntail);
    for (int i = tid; i < WORDS; i += NT) bits[i] = 0;
    if (tid == 0) dup = over = 0;
    for (int j = tid; j < a.K; j += NT) dist_load_entry<T>(a, E, row, x, j);
    __syncthreads();
    // mark this segment's listed tokens; a bit found set already means an id that occurs twice
    for (int j = tid; j < a.K; j += NT) {
        const int id = E.id[j] - e0;
        if (E.id[j] >= 0 && id >= 0 && id < len) {
            const uint32_t bit = 1u << (id & 31);
            if (atomicOr(&bits[id >> 5], bit) & bit) dup = 1;
        }
    }
    const float wm = tok_group<64, TokMax>(s.max_of());
    if (lane == 0) red[wave][0] = wm;
    __syncthreads();
    float m = red[0][0];
#pragma unroll
    for (int k = 1; k < NW; ++k) m = tok_max(m, red[k][0]);
    const TokRef ref = tok_ref(m, a.r.c);
    DistSums sum{0.f, 0.f};
    int chain = -1, nl = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (i * NT < nv) {
            float cs = 0.f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) cs += tok_exp2(__builtin_fmaf(TokElem<T>::get(s.r[i], e), ref.c, -ref.mc));
            bool special = s.vm[i] == ref.meq;
            if (a.bucket) {
                const int at = i * NT + tid;
                const uint8_t by = reinterpret_cast<const uint8_t*>(bits)[VEC == 8 ? at : at >> 1];
                special |= (VEC == 8 ? by : by & (15u << ((at & 1) * 4))) != 0;
            }
            list.push(special, s.r[i], i * NT + tid, true, chain, nl);
            sum.S += special ? 0.f : cs;
        }
    }
    if (nl > SPECIAL && lane == 0) over = 1;
    tok_wave_fence();
    for (; chain >= 0; chain = list.next[chain]) {
        const int at = list.vec(chain) * VEC;
        const uint32_t out = a.bucket ? bits[at >> 5] >> (at & 31) : 0;          // a vector's bits lie in one word
        for (int e = 0; e < VEC; ++e) sum.add(list.template get<T>(chain, e), ref, (out >> e) & 1);
    }
    __syncthreads();
    if (over) {                                              // thousands of elements at the maximum: one by one, read again
        sum = DistSums{0.f, 0.f};
        for (int v = tid; v < nv; v += NT) {
            const u32x4_t r = tok_ld16<T>(x + e0 + (int64_t)v * VEC);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const int at = v * VEC + e;
                sum.add(TokElem<T>::get(r, e), ref, a.bucket && ((bits[at >> 5] >> (at & 31)) & 1));
            }
        }
    }
    if (tid < ntail) {
        const int at = nv * VEC + tid;
        sum.add(s.xt, ref, a.bucket && ((bits[at >> 5] >> (at & 31)) & 1));
    }
    const float S1 = tok_group<64, TokSum>(sum.S), n1 = tok_group<64, TokSum>(sum.n);
    if (lane == 0) {
        red[wave][1] = S1;
        red[wave][2] = n1;
    }
    __syncthreads();
    float S = red[0][1], n = red[0][2], mu = m;
#pragma unroll
    for (int k = 1; k < NW; ++k) {
        S += red[k][1];
        n += red[k][2];
    }
    S *= tok_exp2(-ref.dmax);
    if (__builtin_expect(a.bucket && n + S < DIST_FAR, 0)) {    // the second look at the unlisted elements
        const bool tail = tid < ntail && !((bits[nv * VEC / 32] >> ((nv * VEC + tid) & 31)) & 1);
        float um = tail ? s.xt : -INFINITY;
        dist_unlisted<T, NT>(x + e0, nv, bits, [&](float f) { um = tok_max(um, f); });
        um = tok_group<64, TokMax>(um);
        if (lane == 0) red[wave][0] = um;
        __syncthreads();
        um = red[0][0];
#pragma unroll
        for (int k = 1; k < NW; ++k) um = tok_max(um, red[k][0]);
        const TokRef ru = tok_ref(um, a.r.c);
        sum = DistSums{0.f, 0.f};
        dist_unlisted<T, NT>(x + e0, nv, bits, [&](float f) { sum.add(f, ru, false); });
        if (tail) sum.add(s.xt, ru, false);
        S = tok_group<64, TokSum>(sum.S);
        n = tok_group<64, TokSum>(sum.n);
        if (lane == 0) {
            red[wave][1] = S;
            red[wave][2] = n;
        }
        __syncthreads();
        S = red[0][1];
        n = red[0][2];
#pragma unroll
        for (int k = 1; k < NW; ++k) {
            S += red[k][1];
            n += red[k][2];
        }
        S *= tok_exp2(-ru.dmax);
        if (um > -INFINITY) mu = um;
    }
    if (wave == 0) {
        if (a.nseg > 1) {
            if (lane == 0) a.part[u] = make_float4(mu, n, S, m);
        } else {
            const DistRow d = dist_epilogue(a, E, row, w, m, mu, n, S, dup != 0, lane);
            if (lane == 0) rowd = d;
        }
        // fp64 logarithms take as many registers as the row: this wave gives its part up and reads it again (L2)
        if constexpr (GRAD) s.load(x + e0, nv, ntail);
    }
    __syncthreads();
    if constexpr (GRAD) {
        s.forget();
        const DistRow d = rowd;
        const float f = w * a.T, fB = f * d.B;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (i * NT + tid < nv) {
                float g[VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) g[e] = fB * dist_u(d, a.r.c, TokElem<T>::get(s.r[i], e));
                tok_st16<T>(o + (int64_t)(i * NT + tid) * VEC, TokElem<T>::pack(g));
            }
        }
        if (tid < ntail) o[nv * VEC + tid] = TokElem<T>::put(fB * dist_u(d, a.r.c, s.xt));
        __syncthreads();                                 // the listed tokens' stores follow the row's
        for (int j = tid; j < a.K; j += NT)
            if (E.id[j] >= 0) o[E.id[j]] = TokElem<T>::put(f * dist_l(d, a.r.c, E.x[j], E.p[j]));
    }
}

// Joins the segments of a row: one wave a row
template <typename T> __global__ __launch_bounds__(64) void tok_distill_join_kernel(DistArgs a) {
    __shared__ DistEntries E;
    const int lane = threadIdx.x;
    const int64_t row = a.r.u0 + blockIdx.x;
    const float w = a.w ? a.w[row] : 1.f;
    if (w == 0.f) {
        if (lane == 0) a.loss[row] = 0.f;
        return;
    }
    tok_in<T> x = tok_row<T>(a.r, row);
    for (int j = lane; j < a.K; j += 64) dist_load_entry<T>(a, E, row, x, j);
    const float4* part = a.part + row * a.nseg;
    float m = -INFINITY, mu = -INFINITY;                     // mu: the largest reference of a segment that has anything to sum
    for (int s = 0; s < a.nseg; ++s) {
        const float4 p = part[s];
        m = tok_max(m, p.w);
        if (p.y + p.z != 0.f) mu = tok_max(mu, p.x);
    }
    float S = 0.f, n = 0.f;
    for (int s = 0; s < a.nseg; ++s) {
        const float4 p = part[s];
        if (p.x == mu) {
            n += p.y;
            S += p.z;
        } else if (p.x > -INFINITY && p.y + p.z != 0.f) {
            S += (p.y + p.z) * tok_exp2((p.x - mu) * a.r.c);
        } else {
            S += p.z;
        }
    }
    if (!(mu > -INFINITY)) mu = m;
    __syncthreads();
    dist_epilogue(a, E, row, w, m, mu, n, S, true, lane);
    __syncthreads();
}

// ---- narrow rows: G lanes a row, 8 elements a lane ------------------------------------------------------------------------
// p of the listed tokens goes through LDS (one word an element, NOT_LISTED where none): the lane that owns the element picks
// it up for the sums and the gradient.
constexpr uint32_t NOT_LISTED = 0xffffffffu;
// the gradient of a lane's 8 elements f; words: p of the listed ones
__device__ __forceinline__ void dist_narrow_dx(const DistRow& d, float c, bool live, float fw, const uint32_t* words, float* f) {
    if (__builtin_expect(__ballot(live && d.mu != d.m) != 0, 0)) {    // some row of the wave whose rest has a reference of its own
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t pb = words[e];
            const float g = pb == NOT_LISTED ? d.B * dist_u(d, c, f[e]) : dist_l(d, c, f[e], __uint_as_float(pb));
            f[e] = live ? fw * g : 0.f;
        }
        return;
    }
    const bool none = d.l2S == INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) {                            // one exponential for either kind
        const uint32_t pb = words[e];
        const bool un = pb == NOT_LISTED;
        const float q = tok_exp2(__builtin_fmaf(f[e] - d.m, c, -(un ? d.l2u : d.l2S)));
        const float g = un ? d.B * q : none ? 0.f : __builtin_fmaf(d.A, q, -__uint_as_float(pb));
        f[e] = live ? fw * g : 0.f;
    }
}
struct DistSum {
    double rest, listed, tot, acc;
    float m, mu, s, w;
};

template <typename T, int G, bool GRAD>
__global__ __launch_bounds__(256) void tok_distill_narrow_kernel(DistArgs a) {
    constexpr int RB = 256 / G;
    __shared__ uint32_t buf[256 * 8];                        // a row's words belong to its group of lanes: fences of the wave
    __shared__ DistSum sums[RB];
    __shared__ DistDone done[RB];
    const int gl = threadIdx.x & (G - 1), gr = threadIdx.x / G;
    uint32_t* mine = buf + gr * G * 8;
    const int V = a.r.V, K = a.K;
    const int64_t row = (a.r.u0 + blockIdx.x) * RB + gr;
    const bool there = row < a.r.rows;
    const float w = there ? (a.w ? a.w[row] : 1.f) : 0.f;
    const bool live = there && w != 0.f;
    tok_in<T> x = live ? tok_row<T>(a.r, row) : (tok_in<T>)0;
    float f[8];
    tok_narrow_load<T>(x, V, gl * 8, live, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) mine[gl * 8 + e] = NOT_LISTED;
    tok_wave_fence();
    bool twice = false;
    float s = -INFINITY;
    if (live)
        for (int j = gl; j < K; j += G) {
            const int64_t id = tok_int(a.ids, a.id64, row * K + j);
            if ((uint64_t)id < (uint64_t)V) {
                twice |= atomicExch(&mine[id], 0u) != NOT_LISTED;
                s = tok_max(s, a.t[row * K + j]);
            }
        }
    tok_wave_fence();
    float m = tok_max(tok_max3(tok_max3(f[0], f[1], f[2]), f[3], f[4]), tok_max3(f[5], f[6], f[7]));
    m = tok_group<G, TokMax>(m);
    const TokRef ref = tok_ref(m, a.r.c);
    DistSums un{0.f, 0.f}, li{0.f, 0.f};                     // unlisted, listed (drop mode needs their sum alone)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const bool l = mine[gl * 8 + e] != NOT_LISTED;
        un.add(f[e], ref, l);
        li.add(f[e], ref, !l);
    }
    float S = tok_group<G, TokSum>(un.S) * tok_exp2(-ref.dmax), n = tok_group<G, TokSum>(un.n), mu = m;
    const float Sl = tok_group<G, TokSum>(li.S), nl = tok_group<G, TokSum>(li.n);
    const double sc = (double)tok_exp2(-ref.dmax);
    const bool far = a.bucket && live && n + S < DIST_FAR;
    if (__builtin_expect(__ballot(far) != 0, 0)) {    // some row of the wave: the second look at the unlisted elements
        float um = -INFINITY;
#pragma unroll
        for (int e = 0; e < 8; ++e) um = mine[gl * 8 + e] != NOT_LISTED ? um : tok_max(um, f[e]);
        um = tok_group<G, TokMax>(um);
        const TokRef ru = tok_ref(um, a.r.c);
        DistSums su{0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 8; ++e) su.add(f[e], ru, mine[gl * 8 + e] != NOT_LISTED);
        const float Su = tok_group<G, TokSum>(su.S) * tok_exp2(-ru.dmax), nu = tok_group<G, TokSum>(su.n);
        if (far) {
            S = Su;
            n = nu;
            if (um > -INFINITY) mu = um;
        }
    }
    s = a.bucket ? 0.f : tok_group<G, TokMax>(s);
    if (!(s > -INFINITY)) s = 0.f;
    const bool dup = __ballot(twice) != 0;                   // any row of this wave
    DistTeach te{0.0, 0.0};
    if (live)
        for (int j = gl; j < K; j += G) {
            const int64_t id = tok_int(a.ids, a.id64, row * K + j);
            if ((uint64_t)id < (uint64_t)V) te.add(a.t[row * K + j], s, TokElem<T>::one(x[id]), m, a.r.dinv_t);
        }
    if (__builtin_expect(dup, 0) && live) {
        float more = 0.f;
        for (int j = gl; j < K; j += G) {
            const int64_t id = tok_int(a.ids, a.id64, row * K + j);
            if ((uint64_t)id < (uint64_t)V)
                more += dist_parts(K, a.t[row * K + j], s, [&](int i) { return tok_int(a.ids, a.id64, row * K + i) == id; },
                                   [&](int i) { return a.t[row * K + i]; });
        }
        te.acc += (double)more;
    }
    te.tot = tok_group<G, TokSum>(te.tot);
    te.acc = tok_group<G, TokSum>(te.acc);
    // the fp64 logarithms of all rows of the block by one wave, a row a lane (120,000 rows of 200 bf16 logits, K = 8, tail bucket:
    // 70 us, by each wave for its own rows 89, when both were tried; 73 now, with the rest's own reference)
    if (gl == 0) {
        sums[gr].rest = (double)n + (double)S;
        sums[gr].listed = (double)nl + (double)Sl * sc;
        sums[gr].tot = te.tot;
        sums[gr].acc = te.acc;
        sums[gr].m = m;
        sums[gr].mu = mu;
        sums[gr].s = s;
        sums[gr].w = w;
    }
    __syncthreads();                                         // the marks have been read, too
    if (threadIdx.x < RB) {
        const DistSum q = sums[threadIdx.x];
        const DistDone d = dist_finish(a, q.m, q.mu, q.rest, q.listed, q.tot, q.acc, q.s);
        done[threadIdx.x] = d;
        const int64_t rw = (a.r.u0 + blockIdx.x) * RB + threadIdx.x;
        if (rw < a.r.rows) {
            a.loss[rw] = q.w != 0.f ? (float)((double)q.w * (double)a.T * (double)a.T * d.kl) : 0.f;
            if (a.stat && q.w != 0.f) dist_keep(a.stat, rw, d.d);
        }
    }
    __syncthreads();
    const DistDone r = done[gr];
    if (live && (GRAD || a.pk))
        for (int j = gl; j < K; j += G) {
            const int64_t id = tok_int(a.ids, a.id64, row * K + j);
            if ((uint64_t)id >= (uint64_t)V) continue;
            float p = dist_p(a.t[row * K + j], r.shift);
            if (dup) {                                       // each occurrence has the whole p
                p = 0.f;
                for (int i = 0; i < K; ++i)
                    if (tok_int(a.ids, a.id64, row * K + i) == id) p += dist_p(a.t[row * K + i], r.shift);
            }
            mine[id] = __float_as_uint(p);
            if (a.pk) a.pk[row * K + j] = p;
        }
    tok_wave_fence();
    if constexpr (GRAD) {
        if (there && gl * 8 < V) {
            const float fw = w * a.T;
            dist_narrow_dx(r.d, a.r.c, live, fw, mine + gl * 8, f);
            tok_narrow_store<T>((tok_out<T>)a.dx + row * V, V, gl * 8, f);
        }
    }
}

// Many short rows: a row a lane; the listed tokens are the bits of a 64-bit word, the entries wait in LDS, and so does the
// gradient's row while the listed tokens are put into it.
constexpr int DIST_LANE_K = 16;       // 64 rows' entries in 8 KB of LDS

template <typename T, bool GRAD> __global__ __launch_bounds__(64) void tok_distill_lane_kernel(DistArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint64_t lane_lds[];
    const int V = a.r.V, K = a.K, lane = threadIdx.x;
    T* rows = reinterpret_cast<T*>(lane_lds);
    float* ts = reinterpret_cast<float*>(reinterpret_cast<char*>(lane_lds) + (64 * V * sizeof(T) + 15) / 16 * 16);
    signed char* is = reinterpret_cast<signed char*>(ts + 64 * K);
    const int64_t row0 = (a.r.u0 + blockIdx.x) * 64, row = row0 + lane;
    const int nrow = a.r.rows - row0 < 64 ? (int)(a.r.rows - row0) : 64;
    const bool there = lane < nrow;
    const float w = there ? (a.w ? a.w[row] : 1.f) : 0.f;
    const bool live = w != 0.f;
    for (int i0 = lane; i0 < nrow * K; i0 += 64 * 8) {       // 8 entries a lane under way at once
        int64_t id[8];
        float t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i0 + i * 64 < nrow * K) {
                id[i] = tok_int(a.ids, a.id64, row0 * K + i0 + i * 64);
                t[i] = a.t[row0 * K + i0 + i * 64];
            }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i0 + i * 64 < nrow * K) {
                is[i0 + i * 64] = (uint64_t)id[i] < (uint64_t)V ? (signed char)id[i] : (signed char)-1;
                ts[i0 + i * 64] = t[i];
            }
    }
    tok_stage_rows<T>(a.r, row0, nrow, rows);
    T* x = rows + lane * V;
    TokLane<T> l;
    l.load(x, V, -INFINITY);
    uint64_t in = 0;
    bool dup = false;
    float s = -INFINITY;
    for (int j = 0; live && j < K; ++j) {
        const int id = is[lane * K + j];
        if (id < 0) continue;
        dup |= (in >> id) & 1;
        in |= 1ull << id;
        s = tok_max(s, ts[lane * K + j]);
    }
    if (a.bucket || !(s > -INFINITY)) s = 0.f;
    const float m = l.max_of(V, -INFINITY);
    const TokRef ref = tok_ref(m, a.r.c);
    DistSums un{0.f, 0.f}, li{0.f, 0.f};
    if (a.bucket)
        l.each(V, [&](int e, float f) {
            const bool listed = (in >> e) & 1;
            un.add(f, ref, listed);
            li.add(f, ref, !listed);
        });
    else
        l.each(V, [&](int, float f) { un.add(f, ref, false); });
    const double sc = (double)tok_exp2(-ref.dmax);
    float S = un.S * tok_exp2(-ref.dmax), n = un.n, mu = m;
    const bool far = a.bucket && live && n + S < DIST_FAR;
    if (__builtin_expect(__ballot(far) != 0, 0)) {    // some row of the wave: the second look at the unlisted elements
        float um = -INFINITY;
#pragma unroll 1
        for (int e = 0; e < V; ++e) um = (in >> e) & 1 ? um : tok_max(um, TokElem<T>::one(x[e]));
        const TokRef ru = tok_ref(um, a.r.c);
        DistSums su{0.f, 0.f};
#pragma unroll 1
        for (int e = 0; e < V; ++e) su.add(TokElem<T>::one(x[e]), ru, (in >> e) & 1);
        if (far) {
            S = su.S * tok_exp2(-ru.dmax);
            n = su.n;
            if (um > -INFINITY) mu = um;
        }
    }
    DistTeach te{0.0, 0.0};
    for (int j = 0; live && j < K; ++j) {
        const int id = is[lane * K + j];
        if (id >= 0) te.add(ts[lane * K + j], s, TokElem<T>::one(x[id]), m, a.r.dinv_t);
    }
    if (__builtin_expect(dup, 0)) {
        float more = 0.f;
        for (int j = 0; j < K; ++j) {
            const int id = is[lane * K + j];
            if (id >= 0)
                more += dist_parts(K, ts[lane * K + j], s, [&](int i) { return is[lane * K + i] == id; },
                                   [&](int i) { return ts[lane * K + i]; });
        }
        te.acc += (double)more;
    }
    const DistDone r = dist_finish(a, m, mu, (double)n + (double)S, (double)li.n + (double)li.S * sc, te.tot, te.acc, s);
    if (there) {
        a.loss[row] = live ? (float)((double)w * (double)a.T * (double)a.T * r.kl) : 0.f;
        if (a.stat && live) dist_keep(a.stat, row, r.d);
    }
    const float f = w * a.T, fB = f * r.d.B;
    float g[DIST_LANE_K];                                    // the entries' gradients, the student's row still in LDS
#pragma unroll
    for (int j = 0; j < DIST_LANE_K; ++j) {
        g[j] = 0.f;
        const int id = (GRAD || a.pk) && j < K ? is[lane * K + j] : -1;
        if (id >= 0 && live) {
            float p = 0.f;
            if (!dup) {
                p = dist_p(ts[lane * K + j], r.shift);
            } else {                                         // each occurrence has the whole p
                for (int i = 0; i < K; ++i)
                    if (is[lane * K + i] == id) p += dist_p(ts[lane * K + i], r.shift);
            }
            if (a.pk) a.pk[row * K + j] = p;
            if (!r.none) g[j] = f * __builtin_fmaf(r.d.A, dist_q(r.d, a.r.c, TokElem<T>::one(x[id])), -p);
        }
    }
    if constexpr (GRAD) {
        l.each(V, [&](int, float& v) { v = live ? fB * dist_u(r.d, a.r.c, v) : 0.f; });
        if (there) {
            l.store(x, V);
#pragma unroll
            for (int j = 0; j < DIST_LANE_K; ++j)            // an id that occurs twice is stored twice, the same value
                if (j < K && live && is[lane * K + j] >= 0) x[is[lane * K + j]] = TokElem<T>::put(g[j]);
        }
        tok_wave_fence();
        tok_stage_out<T>(rows, (tok_out<T>)a.dx + row0 * V, nrow * V);
    }
}

// ---- gradient from the saved statistics ------------------------------------------------------------------------------------
struct DistGradArgs {
    TokRows r;
    int64_t ids;
    int id64, K, chunks;
    float T;
    const float *w, *g, *pk;     // g: the gradient of each row's loss
    const float4* stat;
    int64_t dx;
};

template <typename T> __global__ __launch_bounds__(256) void tok_distill_grad_kernel(DistGradArgs a) {
    constexpr int VEC = TokElem<T>::VEC, U = 4;
    const int tid = threadIdx.x;
    const int nvec = a.r.V / VEC, ntail = a.r.V - nvec * VEC;
    const int64_t u = a.r.u0 + blockIdx.x;
    const int64_t row = u / a.chunks;
    const int ch = (int)(u - row * a.chunks);
    const float w = a.w ? a.w[row] : 1.f;
    tok_out<T> o = (tok_out<T>)a.dx + row * a.r.V;
    tok_in<T> x = tok_row<T>(a.r, row);
    const int b0 = ch * 256 * U;
    const bool live = w != 0.f;
    const DistRow d = live ? dist_kept(a.stat, row) : DistRow{0.f, INFINITY, 0.f, 0.f, INFINITY, 0.f};
    const float f = live ? w * a.T * (a.g ? a.g[row] : 1.f) : 0.f, fB = f * d.B;
    u32x4_t r[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int v = b0 + i * 256 + tid;
        r[i] = u32x4_t{0, 0, 0, 0};
        if (live && v < nvec) r[i] = tok_ld16<T>(x + (int64_t)v * VEC);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int v = b0 + i * 256 + tid;
        if (v < nvec) {
            float g[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) g[e] = live ? fB * dist_u(d, a.r.c, TokElem<T>::get(r[i], e)) : 0.f;
            tok_st16<T>(o + (int64_t)v * VEC, TokElem<T>::pack(g));
        }
    }
    const bool last = ch == a.chunks - 1;
    if (last && tid < ntail) {
        const int e = nvec * VEC + tid;
        o[e] = TokElem<T>::put(live ? fB * dist_u(d, a.r.c, TokElem<T>::one(x[e])) : 0.f);
    }
    __syncthreads();                                     // the listed tokens' stores follow the block's own
    if (live) {
        const int64_t lo = (int64_t)b0 * VEC, hi = last ? a.r.V : lo + 256 * U * VEC;
        for (int j = tid; j < a.K; j += 256) {
            const int64_t id = tok_int(a.ids, a.id64, row * a.K + j);
            if (id >= lo && id < hi)
                o[id] = TokElem<T>::put(f * dist_l(d, a.r.c, TokElem<T>::one(x[id]), a.pk[row * a.K + j]));
        }
    }
}

template <typename T, int G> __global__ __launch_bounds__(256) void tok_distill_grad_narrow_kernel(DistGradArgs a) {
    constexpr int RB = 256 / G;
    __shared__ uint32_t buf[256 * 8];
    const int gl = threadIdx.x & (G - 1), gr = threadIdx.x / G;
    uint32_t* mine = buf + gr * G * 8;
    const int V = a.r.V, K = a.K;
    const int64_t r0 = (a.r.u0 + blockIdx.x) * RB;
    const int64_t row = r0 + gr;
    const bool there = row < a.r.rows;
    const float w = there ? (a.w ? a.w[row] : 1.f) : 0.f;
    const bool live = there && w != 0.f;
    float f[8];
    tok_narrow_load<T>(live ? tok_row<T>(a.r, row) : (tok_in<T>)0, V, gl * 8, live, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) mine[gl * 8 + e] = NOT_LISTED;
    __syncthreads();
    if (live)
        for (int j = gl; j < K; j += G) {
            const int64_t id = tok_int(a.ids, a.id64, row * K + j);
            if ((uint64_t)id < (uint64_t)V) mine[id] = __float_as_uint(a.pk[row * K + j]);
        }
    __syncthreads();
    if (there && gl * 8 < V) {
        const DistRow d = live ? dist_kept(a.stat, row) : DistRow{0.f, INFINITY, 0.f, 0.f, INFINITY, 0.f};
        dist_narrow_dx(d, a.r.c, live, live ? w * a.T * (a.g ? a.g[row] : 1.f) : 0.f, mine + gl * 8, f);
        tok_narrow_store<T>((tok_out<T>)a.dx + row * V, V, gl * 8, f);
    }
}

// ---- launchers -------------------------------------------------------------------------------------------------------------
// One pass (loss and gradient from one read) for rows of up to 16384 vectors (1024 threads x 16): 2,000 rows of 50,001 fp32
// logits 182 us, by two launches 243; statistics alone whole up to 8192
constexpr int DIST_ONE_PASS_VEC = 16384;

static TokPlan dist_plan(int64_t V, int dtype) { return tok_plan(V, tok_esize(dtype), 8192); }
static bool dist_one_pass(int64_t V, int dtype) { return V / (16 / tok_esize(dtype)) <= DIST_ONE_PASS_VEC; }

// Workspace of a call: segments a row is cut into (16 bytes each when more than one); 0: the one-pass form (with a gradient),
// which needs no workspace, stat or pk
int64_t tok_distill_segments(int64_t V, int dtype, int grad) {
    if (V <= TOK_NARROW_V) return grad ? 0 : 1;
    if (grad && dist_one_pass(V, dtype)) return 0;
    return dist_plan(V, dtype).nseg;
}

template <typename T, bool GRAD> static void distill_wide(const DistArgs& a, const TokPlan& p, hipStream_t s) {
    const int64_t units = a.r.rows * p.nseg;
    const int nt = p.nt;
    if (p.nt == 64 && p.nv == 2) tok_launch(tok_distill_kernel<T, 64, 2, GRAD>, units, nt, 0, s, a);
    else if (p.nt == 64 && p.nv == 4) tok_launch(tok_distill_kernel<T, 64, 4, GRAD>, units, nt, 0, s, a);
    else if (p.nt == 64) tok_launch(tok_distill_kernel<T, 64, 8, GRAD>, units, nt, 0, s, a);
    else if (p.nv == 4) tok_launch(tok_distill_kernel<T, 256, 4, GRAD>, units, nt, 0, s, a);
    else if (p.nv == 8) tok_launch(tok_distill_kernel<T, 256, 8, GRAD>, units, nt, 0, s, a);
    else if (p.nt == 256) tok_launch(tok_distill_kernel<T, 256, 16, GRAD>, units, nt, 0, s, a);
    else if (p.nt == 512) tok_launch(tok_distill_kernel<T, 512, 16, GRAD>, units, nt, 0, s, a);
    else if constexpr (GRAD) tok_launch(tok_distill_kernel<T, 1024, 16, GRAD>, units, nt, 0, s, a);
}
template <typename T, bool GRAD> static void distill_narrow(const DistArgs& a, hipStream_t s) {
    if (tok_lane_rows(a.r.V, sizeof(T), a.r.rows) && a.K <= DIST_LANE_K) {
        const size_t lds = (64 * a.r.V * sizeof(T) + 15) / 16 * 16 + 64 * a.K * 5;
        tok_launch(tok_distill_lane_kernel<T, GRAD>, (a.r.rows + 63) / 64, 64, lds, s, a);
        return;
    }
    const int G = tok_narrow_lanes(a.r.V);
    const int64_t rb = 256 / G;
    const int64_t units = (a.r.rows + rb - 1) / rb;
    const int nt = 256;
    if (G == 8) tok_launch(tok_distill_narrow_kernel<T, 8, GRAD>, units, nt, 0, s, a);
    else if (G == 16) tok_launch(tok_distill_narrow_kernel<T, 16, GRAD>, units, nt, 0, s, a);
    else if (G == 32) tok_launch(tok_distill_narrow_kernel<T, 32, GRAD>, units, nt, 0, s, a);
    else tok_launch(tok_distill_narrow_kernel<T, 64, GRAD>, units, nt, 0, s, a);
}
template <typename T> static void distill_any(const DistArgs& a, const TokPlan* p, bool grad, hipStream_t s) {
    if (!p) grad ? distill_narrow<T, true>(a, s) : distill_narrow<T, false>(a, s);
    else grad ? distill_wide<T, true>(a, *p, s) : distill_wide<T, false>(a, *p, s);
}
template <typename T> static void distill_grad_any(DistGradArgs a, hipStream_t s) {
    const int V = a.r.V;
    if (V <= TOK_NARROW_V) {
        const int G = tok_narrow_lanes(V);
        const int64_t rb = 256 / G;
        const int64_t units = (a.r.rows + rb - 1) / rb;
        const int nt = 256;
        if (G == 8) tok_launch(tok_distill_grad_narrow_kernel<T, 8>, units, nt, 0, s, a);
        else if (G == 16) tok_launch(tok_distill_grad_narrow_kernel<T, 16>, units, nt, 0, s, a);
        else if (G == 32) tok_launch(tok_distill_grad_narrow_kernel<T, 32>, units, nt, 0, s, a);
        else tok_launch(tok_distill_grad_narrow_kernel<T, 64>, units, nt, 0, s, a);
        return;
    }
    a.chunks = (V / TokElem<T>::VEC + 1023) / 1024;
    tok_launch(tok_distill_grad_kernel<T>, a.r.rows * a.chunks, 256, 0, s, a);
}

// dtype: 0 fp32, 1 bf16, 2 fp16.  dx = 0: loss, stat and pk (for launch_tok_distill_grad).  dx: the gradient too, for a loss
// gradient of 1 a row; stat / pk / ws as tok_distill_segments says.
void launch_tok_distill(uint64_t x, int dtype, int64_t rows, int64_t n1, int64_t s0, int64_t s1, int64_t V, double temperature,
                        uint64_t ids, int id64, uint64_t t, uint64_t w, int K, int bucket, uint64_t loss, uint64_t dx,
                        uint64_t stat, uint64_t pk, uint64_t ws, uint64_t stream) {
    if (rows <= 0) return;
    if (dtype < 0 || dtype > 2) throw std::runtime_error("token operators: unknown logits type");
    if (K < 1 || K > DIST_MAX_K) throw std::runtime_error("tok_distill: 1 to 256 teacher entries a row");
    if (!ids || !t || !loss) throw std::runtime_error("tok_distill: a tensor has no storage");
    DistArgs a{};
    a.r = tok_rows_of(x, rows, n1, s0, s1, V, temperature);
    a.ids = (int64_t)ids;
    a.id64 = id64;
    a.t = as_ptr<const float>(t);
    a.w = as_ptr<const float>(w);
    a.K = K;
    a.bucket = bucket;
    a.T = (float)temperature;
    a.loss = as_ptr<float>(loss);
    a.dx = (int64_t)dx;
    a.stat = as_ptr<float4>(stat);
    a.pk = as_ptr<float>(pk);
    a.nseg = 1;
    const hipStream_t s = as_stream(stream);
    const bool narrow = V <= TOK_NARROW_V, one = narrow || dist_one_pass(V, dtype), grad = dx && one;
    TokPlan p{};
    if (!narrow) {
        p = grad ? tok_plan(V, tok_esize(dtype), DIST_ONE_PASS_VEC) : dist_plan(V, dtype);
        a.nseg = p.nseg;
        a.segvec = p.segvec;
        if (p.nseg > 1 && !ws) throw std::runtime_error("tok_distill: this shape needs a workspace");
        a.part = as_ptr<float4>(ws);
    }
    if (dx && !grad && (!stat || !pk)) throw std::runtime_error("tok_distill: this shape needs the stat and pk buffers");
    if (dtype == 0) distill_any<float>(a, narrow ? nullptr : &p, grad, s);
    else if (dtype == 1) distill_any<bf16_t>(a, narrow ? nullptr : &p, grad, s);
    else distill_any<f16_t>(a, narrow ? nullptr : &p, grad, s);
    if (a.nseg > 1) {
        const int64_t units = rows;
        const int nt = 64;
        if (dtype == 0) tok_launch(tok_distill_join_kernel<float>, units, nt, 0, s, a);
        else if (dtype == 1) tok_launch(tok_distill_join_kernel<bf16_t>, units, nt, 0, s, a);
        else tok_launch(tok_distill_join_kernel<f16_t>, units, nt, 0, s, a);
    }
    if (dx && !grad)
        launch_tok_distill_grad(x, dtype, rows, n1, s0, s1, V, temperature, ids, id64, w, K, 0, stat, pk, dx, stream);
}

// g = 0: a loss gradient of 1 a row
void launch_tok_distill_grad(uint64_t x, int dtype, int64_t rows, int64_t n1, int64_t s0, int64_t s1, int64_t V,
                             double temperature, uint64_t ids, int id64, uint64_t w, int K, uint64_t g, uint64_t stat,
                             uint64_t pk, uint64_t dx, uint64_t stream) {
    if (rows <= 0) return;
    if (dtype < 0 || dtype > 2) throw std::runtime_error("token operators: unknown logits type");
    if (K < 1 || K > DIST_MAX_K) throw std::runtime_error("tok_distill: 1 to 256 teacher entries a row");
    if (!ids || !stat || !pk || !dx) throw std::runtime_error("tok_distill: a tensor has no storage");
    DistGradArgs a{};
    a.r = tok_rows_of(x, rows, n1, s0, s1, V, temperature);
    a.ids = (int64_t)ids;
    a.id64 = id64;
    a.K = K;
    a.T = (float)temperature;
    a.w = as_ptr<const float>(w);
    a.g = as_ptr<const float>(g);
    a.pk = as_ptr<const float>(pk);
    a.stat = as_ptr<const float4>(stat);
    a.dx = (int64_t)dx;
    const hipStream_t s = as_stream(stream);
    if (dtype == 0) distill_grad_any<float>(a, s);
    else if (dtype == 1) distill_grad_any<bf16_t>(a, s);
    else distill_grad_any<f16_t>(a, s);
}
