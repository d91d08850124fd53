// Log-probabilities of chosen tokens, the clipped policy loss and the preference loss over
// logits, forward and backward, for sm_100a.
//
// Per row of logits x[V] with token k:  m = max x,  s = sum exp(x - m),
//   p = x[k] - m - log s                                    (the token's log-probability)
//   dlogits[j] = c * ([j == k] - exp(x[j] - m)/s),  c = upstream gradient * d value / d p
//
// What bounds them is the logits: 4 bytes a value read, 4 written where the gradient is
// wanted.  A loss and its gradient are one kernel that reads a row once: its values stay in
// registers or shared memory between the row's maximum and sum and the gradient's write.  A row that no CTA
// can hold is held by a cluster of up to 8, whose parts' (maximum, sum) are joined through
// distributed shared memory; so are rows that are too few to fill the card.
// The preference loss's slope depends on all rows of its pair, so its gradient is a second
// pass, from the rows' m and s, in reverse order: the rows read last are still in L2.  Small
// pairs do both passes in one cluster each.
// Differences of log-probabilities are formed in double: they decide on which side of a clip border
// a ratio lies, and a float of p's size is off by more than the ratio should be.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cmath>
#include <cstdint>

#include "program.hpp"

namespace cg = cooperative_groups;

namespace ttb {

namespace {

constexpr int kMaxCluster = 8;  // portable cluster size

struct RowOperand {
    const float* p;  // null: absent
    int64_t s0, s1;
    __device__ float at(int64_t i0, int64_t i1) const { return __ldg(p + i0 * s0 + i1 * s1); }
};

struct TokenArgs {
    const float* logits;
    int64_t ls0, ls1;
    const int* tokens;
    int64_t ts0, ts1;
    RowOperand old, adv, ref, g;
    float* y;
    float* dlogits;
    float* stats;   // preference loss: per row {m, 1/s, p - ref}; null otherwise
    float* slopes;  // preference loss: per pair, upstream gradient * d loss / d S(0)
    int* status;
    int64_t rows, n1;
    int V;  // at most 2^30
    int kind;
    float f0, f1, f2;
};

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN propagates
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// Maximum and sum of exp(x - maximum) of part of a row; joins are exact in any order of the
// maxima, and sums are always joined in the same order.  An empty part is (-inf, 0).
struct Part {
    float m, s;
};

// exp(d), d <= 0, as 2^(d log2 e): two instructions instead of a library exp, which made these
// kernels issue-bound (37 instructions a value; now about 10).  Relative error 2^-22.5 from ex2
// and at most 2.25 |d| 2^-24 from rounding d, the product and the constant; results below the
// normal range become 0.  Sums of values use exp_sum below instead.
__device__ __forceinline__ float exp2_part(float d) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(d));
    return e;
}
__device__ __forceinline__ float exp_part(float d) { return exp2_part(d * 1.44269504f); }

// exp(a - b) for the maxima of a part and a whole: 0 for a part of -inf alone
__device__ __forceinline__ float part_weight(float m, float whole) { return m == -INFINITY ? 0.0f : exp_part(m - whole); }
__device__ __forceinline__ float part_weight_exact(float m, float whole) { return m == -INFINITY ? 0.0f : expf(m - whole); }

// What a row's scalars are formed from: the token's logit and the row's operands.
struct RowNumbers {
    float xk, old, adv, ref, g;
};

// A row: its token, where its logits and its gradient lie, and how they lie within 16 bytes.
// Vectors are cut at the logits' 16-byte boundaries, `shift` values before the row's first.
struct Row {
    int64_t row, i0, i1;
    const float* x;
    float* dx;
    int token, shift;
    bool dx_vec;  // the gradient lies alike
    static __device__ void split(const TokenArgs& a, int64_t r, int64_t& i0, int64_t& i1) {
        if (a.rows <= 0x7fffffff) {
            i0 = static_cast<unsigned>(r) / static_cast<unsigned>(a.n1);
            i1 = static_cast<unsigned>(r) % static_cast<unsigned>(a.n1);
        } else {
            i0 = r / a.n1;
            i1 = r % a.n1;
        }
    }
    static __device__ int token_of(const TokenArgs& a, int64_t r) {
        int64_t i0, i1;
        split(a, r, i0, i1);
        return __ldg(a.tokens + i0 * a.ts0 + i1 * a.ts1);
    }
    __device__ Row(const TokenArgs& a, int64_t r) : Row(a, r, token_of(a, r)) {}
    __device__ Row(const TokenArgs& a, int64_t r, int t) : row(r), token(t) {
        split(a, r, i0, i1);
        x = a.logits + i0 * a.ls0 + i1 * a.ls1;
        dx = a.dlogits ? a.dlogits + r * a.V : nullptr;
        shift = static_cast<int>(reinterpret_cast<uintptr_t>(x) / 4 % 4);
        dx_vec = static_cast<int>(reinterpret_cast<uintptr_t>(dx) / 4 % 4) == shift;
    }
};

// Values j .. j+3 of a row, -inf outside it.  `once`: they are not read again soon (evict them
// first).
__device__ __forceinline__ void load_vec(const float* x, int j, int V, bool once, float* v) {
    if (j >= 0 && j <= V - 4) {
        const float4* p = reinterpret_cast<const float4*>(x + j);
        const float4 f = once ? __ldcs(p) : __ldg(p);
        v[0] = f.x;
        v[1] = f.y;
        v[2] = f.z;
        v[3] = f.w;
    } else {
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = j + u >= 0 && j + u < V ? __ldg(x + j + u) : -INFINITY;
    }
}
__device__ __forceinline__ void store_vec(float* x, int j, int V, bool vec, const float* v) {
    if (vec && j >= 0 && j <= V - 4) {
        __stcs(reinterpret_cast<float4*>(x + j), make_float4(v[0], v[1], v[2], v[3]));
    } else {
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (j + u >= 0 && j + u < V) x[j + u] = v[u];
    }
}
// The gradient of values j .. j+3 from their exponentials, over them.
__device__ __forceinline__ void grad_vec(float* v, int j, int token, float scale, float c) {
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] *= scale;
    const int k = token - j;
    if (k >= 0 && k < 4) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (u == k) v[u] += c;
    }
}

// A row that is not computed: padding is 0, a token outside the vocabulary is NaN.  `first`:
// this thread writes the row's scalars; vectors from, from + step, ... of the gradient are its.
__device__ void fill_row(const TokenArgs& a, int64_t row, int token, float* dx, bool first, int from, int step) {
    const float v = token < 0 ? 0.0f : __int_as_float(0x7fc00000);
    if (first) {
        if (token >= 0) a.status[1] = TT_STATUS_BAD_TOKEN;
        if (a.stats) a.stats[3 * row + 2] = v;
        else if (a.y) a.y[row] = v;
    }
    if (!dx || a.stats) return;
    const int out = static_cast<int>(reinterpret_cast<uintptr_t>(dx) / 4 % 4);
    const float f[4] = {v, v, v, v};
    for (int q = from; 4 * q - out < a.V; q += step) store_vec(dx, 4 * q - out, a.V, true, f);
}

__device__ __forceinline__ RowNumbers row_numbers(const TokenArgs& a, const Row& r) {
    auto at = [&](const RowOperand& o) { return o.p ? o.at(r.i0, r.i1) : 0.0f; };
    return RowNumbers{__ldg(r.x + r.token), at(a.old), at(a.adv), at(a.ref), a.kind == TK_PREFERENCE ? 0.0f : at(a.g)};
}

// The token's log-probability.  log s of s = 2^k f, 0.75 <= f < 1.5, is k log 2 (in double) + logf(f):
// |log f| < 0.41, so that float is off by 3e-8 at most, where logf(s) would be by 1e-6.  The
// preference loss, which sums many of them, takes a double log.
__device__ __forceinline__ double token_logp(float xk, Part all) {
    const int bits = __float_as_int(all.s), k = (bits - 0x3f400000) >> 23;
    const double log_s = bits >= 0x00800000 && bits < 0x7f800000
                             ? k * 0.69314718055994530942 + static_cast<double>(logf(__int_as_float(bits - (k << 23))))
                             : static_cast<double>(logf(all.s));  // 0 (a row of -inf), inf, NaN
    return static_cast<double>(xk) - static_cast<double>(all.m) - log_s;
}
__device__ __forceinline__ double token_logp_exact(float xk, Part all) {
    return static_cast<double>(xk) - static_cast<double>(all.m) - log(static_cast<double>(all.s));
}

// The gradient's factor c = g * d value / d p.  Ratios are expf of differences formed in double
// (2 ulp on the slope): the row's data threads wait for this, and two double exponentials in
// a row took longer than the cluster's exchange.
__device__ __forceinline__ float row_slope(const TokenArgs& a, const RowNumbers& k, double p) {
    if (a.kind != TK_POLICY) return k.g;
    const float r = expf(static_cast<float>(p - static_cast<double>(k.old)));
    const float lo = 1.0f - a.f0, hi = 1.0f + a.f1;
    const float plain = r * k.adv, held = (r < lo ? lo : r > hi ? hi : r) * k.adv;
    float slope = plain <= held ? -plain : 0.0f;
    if (plain != plain) slope = plain;  // NaN in the row or its numbers
    if (a.ref.p) slope -= a.f2 * expm1f(static_cast<float>(static_cast<double>(k.ref) - p));
    return slope * k.g;
}

// The row's value, or its stats for the preference loss.
__device__ __forceinline__ void write_value(const TokenArgs& a, int64_t row, const RowNumbers& k, Part all, double p) {
    if (a.stats) {
        a.stats[3 * row] = all.m;
        a.stats[3 * row + 1] = 1.0f / all.s;
        a.stats[3 * row + 2] = static_cast<float>(p - static_cast<double>(k.ref));
        return;
    }
    if (!a.y) return;
    if (a.kind != TK_POLICY) {
        a.y[row] = static_cast<float>(p);
        return;
    }
    const float r = expf(static_cast<float>(p - static_cast<double>(k.old)));
    const float lo = 1.0f - a.f0, hi = 1.0f + a.f1;
    const float plain = r * k.adv, held = (r < lo ? lo : r > hi ? hi : r) * k.adv;
    float value = plain <= held ? -plain : -held;
    if (plain != plain) value = plain;
    if (a.ref.p) {
        const float d = static_cast<float>(static_cast<double>(k.ref) - p);
        value += a.f2 * (expm1f(d) - d);
    }
    a.y[row] = value;
}

__device__ __forceinline__ float warp_max(float v) {  // NaN propagates
    float d;
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(d) : "f"(v));
    return d;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Two float32 operations in one instruction, each rounded as the scalar one.
struct Pair {
    uint64_t v;
};
__device__ __forceinline__ Pair pair(float x, float y) {
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(x), "f"(y));
    return p;
}
__device__ __forceinline__ float2 halves(Pair p) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p.v));
    return f;
}
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}

__device__ __forceinline__ Pair fma(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}

// exp(d) of two d <= 0, for sums without a gradient.  exp2_part's mean error is not 0 (about 4e-8
// with its constant's), which all rows share and the preference loss adds up over a sequence's
// tokens: an answer against an empty one was off by 1.3e-6, four times what it is with these.
// d log2 e = n + f, |f| <= 1/2: n is rounded off by adding 1.5 * 2^23, f is formed by fused
// multiply-adds with log2 e in two floats, 2^f is its interpolant of degree 6 at the Chebyshev
// points of [-1/2, 1/2] (2.5e-9; 7.6e-8 with its roundings, whose mean is 1e-9), and n is added to
// the exponent.  d below -87.3 (-inf: outside the row) counts as that: at most 2^30 terms of
// 2^-126 beside a term of 1.  NaN and infinite maxima are the caller's.
__device__ __forceinline__ Pair exp_sum(Pair d) {
    float2 h = halves(d);
    d = pair(fmaxf(h.x, -87.3f), fmaxf(h.y, -87.3f));
    const Pair log2e = pair(1.44269502f, 1.44269502f), rest = pair(1.92596300e-8f, 1.92596300e-8f);
    const Pair magic = pair(12582912.0f, 12582912.0f), n = fma(d, log2e, magic);
    const Pair f = fma(d, rest, fma(d, log2e, fma(n, pair(-1.0f, -1.0f), magic)));
    Pair y = pair(1.54614449e-4f, 1.54614449e-4f);
    const float c[6] = {1.0f, 0.693147182f, 0.240226507f, 0.0555032715f, 0.00961805694f, 0.00134004280f};
#pragma unroll
    for (int q = 5; q >= 0; --q) y = fma(y, f, pair(c[q], c[q]));
    const float2 a = halves(y), e = halves(n);
    return pair(__int_as_float(__float_as_int(a.x) + (__float_as_int(e.x) << 23)),
                __int_as_float(__float_as_int(a.y) + (__float_as_int(e.y) << 23)));
}

// The part of a warp from its threads' values: v becomes exp(v - maximum).  Maxima and sums
// run in four chains a thread: one chain of 32 dependent operations cost more than their number.
// EXACT: for sums without a gradient; v is left as it was.
template <int NV, bool EXACT>
__device__ __forceinline__ Part warp_part(float (*v)[4]) {
    float m4[4] = {v[0][0], v[0][1], v[0][2], v[0][3]};
#pragma unroll
    for (int q = 1; q < NV; ++q)
#pragma unroll
        for (int u = 0; u < 4; ++u) m4[u] = max_nan(m4[u], v[q][u]);
    const float m = warp_max(max_nan(max_nan(m4[0], m4[1]), max_nan(m4[2], m4[3])));
    const float from = m == -INFINITY ? 0.0f : m;
    const Pair shift = pair(-from, -from), log2e = pair(1.44269504f, 1.44269504f);
    Pair s0 = pair(0.0f, 0.0f), s1 = s0;
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        if (EXACT) {
            s0 = s0 + exp_sum(pair(v[q][0], v[q][1]) + shift);
            s1 = s1 + exp_sum(pair(v[q][2], v[q][3]) + shift);
            continue;
        }
        const float2 a = halves((pair(v[q][0], v[q][1]) + shift) * log2e), b = halves((pair(v[q][2], v[q][3]) + shift) * log2e);
        v[q][0] = exp2_part(a.x);
        v[q][1] = exp2_part(a.y);
        v[q][2] = exp2_part(b.x);
        v[q][3] = exp2_part(b.y);
        s0 = s0 + pair(v[q][0], v[q][1]);
        s1 = s1 + pair(v[q][2], v[q][3]);
    }
    const float2 s = halves(s0 + s1);
    const float sum = warp_sum(s.x + s.y);
    return Part{m, EXACT ? fmaf(0.0f, from, sum) : sum};  // a maximum of NaN or inf: NaN
}

// Joins N parts (a multiple of 32 or less than 32), the same in every thread of the warp.
template <bool EXACT>
__device__ __forceinline__ Part join_parts(const Part* parts, int n, int l) {
    Part all{-INFINITY, 0.0f};
    for (int q = l; q < n; q += 32) all.m = max_nan(all.m, parts[q].m);
    all.m = warp_max(all.m);
    for (int q = l; q < n; q += 32) all.s += parts[q].s * (EXACT ? part_weight_exact(parts[q].m, all.m) : part_weight(parts[q].m, all.m));
    all.s = warp_sum(all.s);
    return all;
}

// Hands a warp's part to every CTA of a cluster (lane q < size to CTA q), or to its own CTA.
struct Parts {
    Part of[kMaxCluster * 8];
};
__device__ __forceinline__ void hand_part(Parts& sh, int size, int slot, int l, Part part) {
    if (size == 1) {
        if (l == 0) sh.of[slot] = part;
        __syncthreads();
    } else {
        cg::cluster_group cl = cg::this_cluster();
        if (l < size) cl.map_shared_rank(&sh, l)->of[slot] = part;
        cl.sync();
    }
}

// ---- short rows: a warp holds a row of at most 128*NV values, 8 rows a CTA.  Without a gradient a
// row may be longer: the warp walks it, joining maximum and sum as it goes: 8192 rows of 16384, a fifth
// of them padding, take 84 us (5.0 TB/s; the rows are 1.4 rounds of the card's warps).  A CTA a row took
// 90, a warp that loads ahead of its sums 88.
template <int NV, bool GRAD>
__global__ void __launch_bounds__(256, NV == 16 ? 2 : GRAD || NV == 8 ? 4 : 5) token_warp_kernel(TokenArgs a) {
    const int l = threadIdx.x & 31;
    const int64_t index = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    if (index >= a.rows) return;
    const Row r(a, index);
    if (r.token < 0 || r.token >= a.V) {
        fill_row(a, r.row, r.token, r.dx, l == 0, l, 32);
        return;
    }
    const RowNumbers k = row_numbers(a, r);
    float v[NV][4];
#pragma unroll
    for (int q = 0; q < NV; ++q) load_vec(r.x, 4 * (l + 32 * q) - r.shift, a.V, GRAD, v[q]);
    Part all = warp_part<NV, !GRAD>(v);
    if constexpr (!GRAD) {
        for (int j = 128 * NV - r.shift; j < a.V; j += 128 * NV) {
#pragma unroll
            for (int q = 0; q < NV; ++q) load_vec(r.x, j + 4 * (l + 32 * q), a.V, false, v[q]);
            const Part next = warp_part<NV, true>(v);
            const float m = max_nan(all.m, next.m);
            all.s = all.s * part_weight_exact(all.m, m) + next.s * part_weight_exact(next.m, m);
            all.m = m;
        }
    }
    const double p = GRAD ? token_logp(k.xk, all) : token_logp_exact(k.xk, all);
    if (l == 0) write_value(a, r.row, k, all, p);
    if (!GRAD) return;
    const float c = row_slope(a, k, p);
    const float scale = -c / all.s;  // (a NaN row: the sum is NaN; one of -inf: 0)
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        const int j = 4 * (l + 32 * q) - r.shift;
        grad_vec(v[q], j, r.token, scale, c);
        store_vec(r.dx, j, a.V, r.dx_vec, v[q]);
    }
}

// ---- values without a gradient, and rows longer than a cluster can hold: every CTA walks its
// share of a row once, joining maximum and sum as it goes; for the gradient it reads it a second
// time (mostly from L2, latest first).  Few rows are shared by a cluster: 8 rows of 131072 take 10 us on
// 8 CTAs each, a launch, three loads' latencies and the cluster's exchange.
constexpr int kStream = 256, kStreamVec = 8;
constexpr int kWalk = 4096;  // vectors of the longest row that one warp walks

template <bool GRAD>
__global__ void __launch_bounds__(kStream, 4) token_stream_kernel(TokenArgs a) {
    __shared__ Parts sh;
    const int tid = threadIdx.x, l = tid & 31, warp = tid >> 5;
    cg::cluster_group cl = cg::this_cluster();
    const int size = static_cast<int>(cl.num_blocks()), rank = static_cast<int>(cl.block_rank());
    const Row r(a, blockIdx.x / size);
    if (r.token < 0 || r.token >= a.V) {  // (the whole cluster leaves)
        fill_row(a, r.row, r.token, r.dx, tid == 0 && rank == 0, rank * kStream + tid, size * kStream);
        return;
    }
    if (size > 1) cl.barrier_arrive();  // every CTA runs before another writes to it
    const RowNumbers k = row_numbers(a, r);
    const int vectors = (a.V + r.shift + 3) / 4, share = (vectors + size - 1) / size;
    const int begin = min(vectors, rank * share), end = min(vectors, begin + share);
    Part t{-INFINITY, 0.0f};
    for (int q0 = begin + tid; q0 < end; q0 += kStreamVec * kStream) {
        float v[kStreamVec][4];
#pragma unroll
        for (int q = 0; q < kStreamVec; ++q) {
            const bool in = q0 + q * kStream < end;
            load_vec(r.x, in ? 4 * (q0 + q * kStream) - r.shift : 0, in ? a.V : 0, false, v[q]);
        }
        float m = t.m;
#pragma unroll
        for (int q = 0; q < kStreamVec; ++q)
#pragma unroll
            for (int u = 0; u < 4; ++u) m = max_nan(m, v[q][u]);
        const float from = m == -INFINITY ? 0.0f : m;
        const Pair shift = pair(-from, -from);
        Pair s0 = pair(0.0f, 0.0f), s1 = s0;
#pragma unroll
        for (int q = 0; q < kStreamVec; ++q) {
            s0 = s0 + exp_sum(pair(v[q][0], v[q][1]) + shift);
            s1 = s1 + exp_sum(pair(v[q][2], v[q][3]) + shift);
        }
        const float2 s = halves(s0 + s1);
        t.s = t.s * part_weight_exact(t.m, from) + fmaf(0.0f, from, s.x + s.y);  // a maximum of NaN or inf: NaN
        t.m = m;
    }
    Part w;
    w.m = warp_max(t.m);
    w.s = warp_sum(t.s * part_weight_exact(t.m, w.m));
    if (size > 1) cl.barrier_wait();
    hand_part(sh, size, rank * (kStream / 32) + warp, l, w);
    if (!GRAD && (warp > 0 || rank > 0)) return;
    const Part all = join_parts<true>(sh.of, size * (kStream / 32), l);
    const double p = token_logp_exact(k.xk, all);
    if (l == 0 && rank == 0 && warp == 0) write_value(a, r.row, k, all, p);
    if (!GRAD) return;
    const float c = row_slope(a, k, p);
    const float scale = -c / all.s;
    for (int q = end - 1 - tid; q >= begin; q -= kStream) {
        float v[4];
        const int j = 4 * q - r.shift;
        load_vec(r.x, j, a.V, true, v);
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = exp_part(v[u] - all.m);
        grad_vec(v, j, r.token, scale, c);
        store_vec(r.dx, j, a.V, r.dx_vec, v);
    }
}

// ---- loss and gradient of rows that a cluster holds.  Clusters walk the rows.  In each CTA G data
// threads hold NV vectors of its share of a row in shared memory (they come by cp.async; a thread
// reads back only what it copied itself) and one more warp joins the parts of the CTA's warps
// and of the cluster's CTAs and forms the row's scalars.  The data threads work on two rows at a
// time: while the scalars of row n are formed they find the maximum and the exponentials of row
// n + 1, and row n + 2 is on its way; then they scale row n and write it.  So neither the
// cluster's exchange nor the scalars' latency is waited for (a form that waited took 5 us a
// row where the bytes take 3).
//   data:  part(n + 1) -> parts full(n + 1) | scalars full(n) -> scale and write row n, fetch n + 3
//   join:  info(n + 4), parts full(n) -> exchange -> scalars(n) -> scalars full(n)
// What bounds it besides the bytes is the instructions a row costs on top of its values, so warps
// whose vectors all lie inside the row move them without checks.
// Clusters of 4 (71 run at a time: 284 of the 296 places) take 336 to 360 us for 8192 rows of 32768 with a
// ninth of them padding (5.7 to 5.3 TB/s, by box), 164 to 168 us for 4096 of 32001 (5.5 to 5.4); clusters of 6 147 us
// for 2177 of 50001 (5.0).
struct RowInfo {
    const float* x;
    float* dx;
    int64_t row;
    int token, shift;
    bool dx_vec;
};
constexpr int kStages = 3, kInfos = 8;

// Barriers between the data threads and the joining warp, one id per parity of the row: a fast
// warp may be one row ahead of a slow one, never two.
template <int N>
__device__ __forceinline__ void named_arrive(int id) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(N) : "memory"); }
template <int N>
__device__ __forceinline__ void named_sync(int id) { asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(N) : "memory"); }

// The exchange of a cluster's parts: each CTA's joining warp writes its part into every CTA's
// shared memory with st.async, which also counts the bytes on that CTA's mbarrier, and waits for
// its own to have all of them.  (A cluster barrier instead held every warp of the cluster to the
// slowest: 3.4 us a row and SM where the bytes take 3.0.)  The wait is bounded: about 2 s, or
// until another kernel of the program gave up; then status word 0 has a code and the rows' results
// are wrong.  The cluster leaves together, so that nobody writes to a CTA that has left.
constexpr int kTimeout = 0x500;
constexpr long long kWaitBudget = 4000000000LL;  // SM cycles
__device__ __forceinline__ void exchange_expect(uint32_t bar, int bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void exchange_send(uint32_t dst, uint32_t bar, int cta, Part part) {
    const uint64_t v = static_cast<uint64_t>(__float_as_uint(part.s)) << 32 | __float_as_uint(part.m);
    asm volatile(
        "{\n\t.reg .b32 d, b;\n\t"
        "mapa.shared::cluster.u32 d, %0, %2;\n\t"
        "mapa.shared::cluster.u32 b, %1, %2;\n\t"
        "st.async.shared::cluster.mbarrier::complete_tx::bytes.b64 [d], %3, [b];\n\t}"
        ::"r"(dst), "r"(bar), "r"(cta), "l"(v) : "memory");
}
__device__ __forceinline__ bool exchange_wait(uint32_t bar, uint32_t parity, int* status) {
    const long long t0 = clock64();
    for (uint32_t polls = 1;; ++polls) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done) : "r"(bar), "r"(parity) : "memory");
        if (done) return true;
        if ((polls & 255) == 0 && *reinterpret_cast<volatile int*>(status) != 0) return false;
        if (clock64() - t0 > kWaitBudget) {
            atomicCAS(status, 0, kTimeout);
            return false;
        }
    }
}

template <int G, int NV>
__global__ void __launch_bounds__(G + 32, 512 / G) token_grad_kernel(TokenArgs a, int clusters) {
    constexpr int N = G + 32, FULL = 1, SCALARS = 3;  // barrier ids (+ parity)
    extern __shared__ __align__(16) float ring[];     // [stage][vector][thread][4]
    __shared__ Part warp_parts[2][G / 32], cta_parts[2][kMaxCluster];
    __shared__ float3 scalars[2];  // m, -c/s, c
    __shared__ RowInfo infos[kInfos];
    __shared__ __align__(8) uint64_t bars[2];  // the exchange's mbarriers, by parity of the computed rows
    cg::cluster_group cl = cg::this_cluster();
    const int size = static_cast<int>(cl.num_blocks()), rank = static_cast<int>(cl.block_rank());
    const int tid = threadIdx.x, l = tid & 31, warp = tid >> 5;
    const int64_t first = blockIdx.x / size;
    const int count = static_cast<int>((a.rows - first + clusters - 1) / clusters);  // this cluster's rows
    auto computed = [&](const RowInfo& r) { return r.token >= 0 && r.token < a.V; };

    if (warp == G / 32) {  // ---- the joining warp
        // lane q keeps operand q of the rows ahead: the token's logit, old, advantage, ref, g.  Tokens are
        // loaded a row earlier still: waiting for them here made this warp the slowest part.
        auto token = [&](int n) { return n < count ? Row::token_of(a, first + static_cast<int64_t>(n) * clusters) : -1; };
        auto look = [&](int n, int tok) {
            if (n >= count) return 0.0f;
            const Row r(a, first + static_cast<int64_t>(n) * clusters, tok);
            if (l == 0) infos[n % kInfos] = RowInfo{r.x, r.dx, r.row, r.token, r.shift, r.dx_vec};
            const RowOperand o = l == 1 ? a.old : l == 2 ? a.adv : l == 3 ? a.ref : l == 4 ? a.g : RowOperand{nullptr, 0, 0};
            if (r.token < 0 || r.token >= a.V) return 0.0f;
            return l == 0 ? __ldg(r.x + r.token) : o.p ? o.at(r.i0, r.i1) : 0.0f;
        };
        float ahead[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) ahead[q] = look(q, token(q));
        int tok = token(4);
        if (l == 0 && size > 1) {
            for (uint64_t& b : bars)
                asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(&b))) : "memory");
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncthreads();
        if (size > 1) cl.sync();  // every CTA runs, with its mbarriers, before another writes to it
        unsigned rows_done = 0;   // computed rows so far
        bool failed = false;
        for (int n = 0; n < count; ++n) {
            const int p = n & 1;
            const RowInfo r = infos[n % kInfos];
            const float mine = ahead[0];
            ahead[0] = ahead[1];
            ahead[1] = ahead[2];
            ahead[2] = ahead[3];
            ahead[3] = look(n + 4, tok);
            tok = token(n + 5);
            named_sync<N>(FULL + p);
            Part all;
            RowNumbers k;
            double logp = 0.0;
            if (computed(r)) {  // (the same for the whole cluster)
                all = join_parts<false>(warp_parts[p], G / 32, l);
                if (size > 1) {
                    const int x = rows_done & 1;
                    const uint32_t bar = static_cast<uint32_t>(__cvta_generic_to_shared(&bars[x]));
                    if (l == 0) exchange_expect(bar, size * static_cast<int>(sizeof(Part)));
                    if (l < size) exchange_send(static_cast<uint32_t>(__cvta_generic_to_shared(&cta_parts[x][rank])), bar, l, all);
                    if (!failed) failed = !exchange_wait(bar, rows_done >> 1 & 1, a.status);
                    failed = __any_sync(0xffffffffu, failed);
                    all = join_parts<false>(cta_parts[x], size, l);
                    ++rows_done;
                }
                k.xk = __shfl_sync(0xffffffffu, mine, 0);
                k.old = __shfl_sync(0xffffffffu, mine, 1);
                k.adv = __shfl_sync(0xffffffffu, mine, 2);
                k.ref = __shfl_sync(0xffffffffu, mine, 3);
                k.g = __shfl_sync(0xffffffffu, mine, 4);
                if (a.kind == TK_POLICY) logp = token_logp(k.xk, all);
                const float c = row_slope(a, k, logp);
                if (l == 0) scalars[p] = make_float3(all.m, -c / all.s, c);
            }
            __syncwarp();
            named_arrive<N>(SCALARS + p);
            if (l == 0 && rank == 0 && computed(r))  // nobody waits for it
                write_value(a, r.row, k, all, a.kind == TK_POLICY ? logp : token_logp(k.xk, all));
        }
        __syncwarp();
        if (size > 1) cl.sync();
        return;
    }

    // ---- the data threads
    const int v0 = 4 * (rank * NV * G + tid);  // this thread's first value, its vectors 4*G apart
    const int lo = v0 - 4 * l, hi = v0 + 4 * (31 - l) + 4 * (NV - 1) * G;  // the warp's first and last vector
    const uint32_t mine = static_cast<uint32_t>(__cvta_generic_to_shared(ring)) + tid * 16;
    auto inside = [&](const RowInfo& r) { return lo >= r.shift && hi - r.shift <= a.V - 4; };
    // A row has two vectors at most that it does not fill, its first and its last: calls f(q, u) for
    // the values of those that are this thread's.
    auto ends = [&](const RowInfo& r, int j0, auto f) {
        if (j0 < 0) {
            for (int u = -j0; u < 4; ++u) f(0, u);
        }
        const int left = (a.V + r.shift) & 3, k = a.V - left - j0;  // the last vector's values, its place
        if (left != 0 && k >= 0 && k / 4 % G == 0 && k / 4 / G < NV) {
            for (int u = 0; u < left; ++u) f(k / 4 / G, u);
        }
    };
    auto fetch = [&](int n) {
        const RowInfo r = infos[n % kInfos];
        if (n < count && computed(r)) {
            const int j0 = v0 - r.shift;
            const uint32_t to = mine + (n % kStages) * NV * G * 16;
            const float* x = r.x + j0;
            if (inside(r)) {
#pragma unroll
                for (int q = 0; q < NV; ++q)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + q * G * 16), "l"(x + 4 * q * G) : "memory");
            } else {
#pragma unroll
                for (int q = 0; q < NV; ++q)
                    if (j0 + 4 * q * G >= 0 && j0 + 4 * q * G <= a.V - 4)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + q * G * 16), "l"(x + 4 * q * G) : "memory");
                ends(r, j0, [&](int q, int u) {
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + q * G * 16 + 4 * u), "l"(x + 4 * q * G + u) : "memory");
                });
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto slot = [&](int n, int q) { return reinterpret_cast<float4*>(ring + (((n % kStages) * NV + q) * G + tid) * 4); };
    // the row's exponentials over its values, this warp's part of the row; returns the warp's maximum
    auto part = [&](int n) {
        const RowInfo r = infos[n % kInfos];
        float m = 0.0f;
        if (computed(r)) {
            float v[NV][4];
#pragma unroll
            for (int q = 0; q < NV; ++q) {
                const float4 f = *slot(n, q);
                v[q][0] = f.x;
                v[q][1] = f.y;
                v[q][2] = f.z;
                v[q][3] = f.w;
            }
            if (!inside(r)) {
                const int j0 = v0 - r.shift;
#pragma unroll
                for (int q = 0; q < NV; ++q)
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        if (static_cast<unsigned>(j0 + 4 * q * G + u) >= static_cast<unsigned>(a.V)) v[q][u] = -INFINITY;
            }
            const Part own = warp_part<NV, false>(v);
#pragma unroll
            for (int q = 0; q < NV; ++q) *slot(n, q) = make_float4(v[q][0], v[q][1], v[q][2], v[q][3]);
            if (l == 0) warp_parts[n & 1][warp] = own;
            m = own.m;
        }
        __syncwarp();
        named_arrive<N>(FULL + (n & 1));
        return m;
    };
    __syncthreads();  // the first rows' infos
    fetch(0);
    fetch(1);
    fetch(2);
    if (size > 1) cl.sync();
    asm volatile("cp.async.wait_group 2;" ::: "memory");
    float own = part(0);
    for (int n = 0; n < count; ++n) {
        float next = 0.0f;
        if (n + 1 < count) {
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            next = part(n + 1);
        }
        named_sync<N>(SCALARS + (n & 1));
        const RowInfo r = infos[n % kInfos];
        const bool real = computed(r);
        if (real) {
            const float3 f = scalars[n & 1];
            const float scale = f.y * part_weight(own, f.x);  // (a NaN row: the sum is NaN; one of -inf: 0)
            const int j0 = v0 - r.shift;
            const int k = r.token - j0;  // the token's place among this thread's vectors
            const bool here = k >= 0 && k < 4 * NV * G && k / 4 % G == 0;
            const bool in = inside(r);
            float* dx = r.dx + j0;
#pragma unroll
            for (int q = 0; q < NV; ++q) {
                float4 e = *slot(n, q);
                const float2 ex = halves(pair(e.x, e.y) * pair(scale, scale)), ez = halves(pair(e.z, e.w) * pair(scale, scale));
                e = make_float4(ex.x, ex.y, ez.x, ez.y);
                if (here && k / 4 == q * G) (k % 4 == 0 ? e.x : k % 4 == 1 ? e.y : k % 4 == 2 ? e.z : e.w) += f.z;
                const int j = j0 + 4 * q * G;
                if (!r.dx_vec) {  // the logits are a view that lies differently: value by value
                    const float v[4] = {e.x, e.y, e.z, e.w};
                    store_vec(r.dx, j, a.V, false, v);
                } else if (in || (j >= 0 && j <= a.V - 4)) {
                    __stcs(reinterpret_cast<float4*>(dx + 4 * q * G), e);
                } else {
                    *slot(n, q) = e;
                }
            }
            if (!in && r.dx_vec) ends(r, j0, [&](int q, int u) { dx[4 * q * G + u] = reinterpret_cast<const float*>(slot(n, q))[u]; });
        } else {
            fill_row(a, r.row, r.token, r.dx, tid == 0 && rank == 0, rank * G + tid, size * G);
        }
        own = next;
        fetch(n + 3);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();
    if (size > 1) cl.sync();  // nobody writes to a CTA that has left
}

// ---- preference loss: the rows' stats, the pairs, the rows again.  8 pairs of 2x512x16384 take 84, 4 and
// 146 us: the gradient's pass runs at the copy bandwidth.  A pair's loss and slope
// from S(0) - S(1), by one thread.
__device__ __forceinline__ float pair_value(const TokenArgs& a, int64_t n, double diff, bool write) {
    const double beta = a.f0, eps = a.f1, z = beta * diff;
    const double e = exp(-fabs(z)), soft = log1p(e);  // soft = -log sigmoid(|z|)
    // (eps = 0 drops its term: an impossible rejected answer has z = inf and loss 0)
    if (write && a.y) a.y[n] = static_cast<float>(soft + (z < 0.0 ? -z * (1.0 - eps) : z == z && eps == 0.0 ? 0.0 : z * eps));
    if (!a.dlogits) return 0.0f;
    const double up = 1.0 / (1.0 + e), down = e / (1.0 + e);  // sigmoid(|z|), sigmoid(-|z|)
    const double pos = z < 0.0 ? down : up, neg = z < 0.0 ? up : down;
    return static_cast<float>(static_cast<double>(a.g.at(n, 0)) * beta * (eps * pos - (1.0 - eps) * neg));
}

// One CTA per pair, from the rows' stats.
constexpr int kPair = 256;
__global__ void __launch_bounds__(kPair) preference_pair_kernel(TokenArgs a) {
    __shared__ double sh[kPair / 32];
    const int64_t n = blockIdx.x, T = a.n1 / 2;
    double v = 0.0;
    for (int64_t t = threadIdx.x; t < T; t += kPair) {
        const float* st = a.stats + 3 * (n * a.n1 + t);
        v += static_cast<double>(st[2]) - static_cast<double>(st[3 * T + 2]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int w = 1; w < kPair / 32; ++w) v += sh[w];
    const float slope = pair_value(a, n, v, true);
    if (a.slopes) a.slopes[n] = slope;
}

// The gradient of a row from its stats, by one warp.
__device__ __forceinline__ void row_gradient(const TokenArgs& a, const Row& r, float c, int l) {
    constexpr int NV = 4;
    if (r.token < 0 || r.token >= a.V) {
        const float f = r.token < 0 ? 0.0f : __int_as_float(0x7fc00000), v[4] = {f, f, f, f};
        const int out = static_cast<int>(reinterpret_cast<uintptr_t>(r.dx) / 4 % 4);
        for (int j = 4 * l - out; j < a.V; j += 128) store_vec(r.dx, j, a.V, true, v);
        return;
    }
    const float m = __ldcg(a.stats + 3 * r.row), scale = -c * __ldcg(a.stats + 3 * r.row + 1);
    for (int j = -r.shift; j < a.V; j += 128 * NV) {
        float v[NV][4];
#pragma unroll
        for (int q = 0; q < NV; ++q) load_vec(r.x, j + 4 * (l + 32 * q), a.V, true, v[q]);
#pragma unroll
        for (int q = 0; q < NV; ++q) {
            const int at = j + 4 * (l + 32 * q);
#pragma unroll
            for (int u = 0; u < 4; ++u) v[q][u] = exp_part(v[q][u] - m);
            grad_vec(v[q], at, r.token, scale, c);
            store_vec(r.dx, at, a.V, r.dx_vec, v[q]);
        }
    }
}

// A pair in one cluster and one launch: its warps walk the pair's rows, the CTAs' sums of p - ref are
// joined, and each warp walks its rows again, latest first, for the gradient.  3 pairs of 2x37x257: 14 us in a
// stream that is flushed before it, 10 us a call; latency.
constexpr int kPairCluster = 8;
template <int NV>
__global__ void __launch_bounds__(256, 4) preference_cluster_kernel(TokenArgs a) {
    __shared__ double warp_sums[8], cta_sums[kPairCluster];
    __shared__ float sh_slope;
    cg::cluster_group cl = cg::this_cluster();
    cl.barrier_arrive();  // every CTA runs before another writes to it
    const int rank = static_cast<int>(cl.block_rank()), l = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t n = blockIdx.x / kPairCluster, T = a.n1 / 2;
    const int first = rank * 8 + warp, step = kPairCluster * 8;
    double sum = 0.0;
    int64_t i = first;
    for (; i < a.n1; i += step) {
        const Row r(a, n * a.n1 + i);
        if (r.token < 0 || r.token >= a.V) {
            fill_row(a, r.row, r.token, r.dx, l == 0, l, 32);
            if (r.token >= 0) sum = __longlong_as_double(0x7ff8000000000000ll);
            continue;
        }
        const RowNumbers k = row_numbers(a, r);
        Part all{-INFINITY, 0.0f};
        for (int j = -r.shift; j < a.V; j += 128 * NV) {
            float v[NV][4];
#pragma unroll
            for (int q = 0; q < NV; ++q) load_vec(r.x, j + 4 * (l + 32 * q), a.V, false, v[q]);
            const Part next = warp_part<NV, true>(v);
            const float m = max_nan(all.m, next.m);
            all.s = all.s * part_weight_exact(all.m, m) + next.s * part_weight_exact(next.m, m);
            all.m = m;
        }
        const double diff = token_logp_exact(k.xk, all) - static_cast<double>(k.ref);
        sum += i < T ? diff : -diff;
        if (l == 0 && a.dlogits) write_value(a, r.row, k, all, diff + static_cast<double>(k.ref));
    }
    if (l == 0) warp_sums[warp] = sum;
    __syncthreads();
    cl.barrier_wait();
    if (threadIdx.x < kPairCluster) {
        double v = 0.0;
        for (int w = 0; w < 8; ++w) v += warp_sums[w];
        *cl.map_shared_rank(&cta_sums[rank], static_cast<int>(threadIdx.x)) = v;
    }
    cl.sync();
    if (threadIdx.x == 0) {
        double v = 0.0;
        for (int q = 0; q < kPairCluster; ++q) v += cta_sums[q];
        sh_slope = pair_value(a, n, v, rank == 0);
    }
    if (!a.dlogits) return;
    __syncthreads();
    const float slope = sh_slope;
    for (i -= step; i >= 0; i -= step) {
        row_gradient(a, Row(a, n * a.n1 + i), i < T ? slope : -slope, l);  // (the warp's own stats, written by lane 0 above)
    }
}

// The preference loss's gradient from the rows' stats, a warp a row: many short rows, which leave most of a CTA
// idle (1000 pairs of 2x64x300 133 us, 498 with a CTA a row; 768 rows of 1000 20 against 15).
__global__ void __launch_bounds__(256) preference_grad_rows_kernel(TokenArgs a) {
    const int64_t index = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    if (index >= a.rows) return;
    const Row r(a, a.rows - 1 - index);
    const float slope = __ldg(a.slopes + r.i0);
    row_gradient(a, r, r.i1 < a.n1 / 2 ? slope : -slope, threadIdx.x & 31);
}

// The same of longer or few rows: a CTA takes kGradVec*kGrad vectors of a row.
constexpr int kGrad = 256, kGradVec = 4;
__global__ void __launch_bounds__(kGrad) preference_grad_kernel(TokenArgs a, int per_row) {
    const Row r(a, a.rows - 1 - blockIdx.x / per_row);
    const int q0 = static_cast<int>(blockIdx.x % per_row) * kGradVec * kGrad + threadIdx.x;
    if (r.token < 0 || r.token >= a.V) {
        const float f = r.token < 0 ? 0.0f : __int_as_float(0x7fc00000), v[4] = {f, f, f, f};
#pragma unroll
        for (int q = 0; q < kGradVec; ++q) store_vec(r.dx, 4 * (q0 + q * kGrad) - r.shift, a.V, r.dx_vec, v);
        return;
    }
    float v[kGradVec][4];
#pragma unroll
    for (int q = 0; q < kGradVec; ++q) load_vec(r.x, 4 * (q0 + q * kGrad) - r.shift, a.V, true, v[q]);
    const float m = __ldg(a.stats + 3 * r.row), slope = __ldg(a.slopes + r.i0), c = r.i1 < a.n1 / 2 ? slope : -slope;
    const float scale = -c * __ldg(a.stats + 3 * r.row + 1);
#pragma unroll
    for (int q = 0; q < kGradVec; ++q) {
        const int j = 4 * (q0 + q * kGrad) - r.shift;
#pragma unroll
        for (int u = 0; u < 4; ++u) v[q][u] = exp_part(v[q][u] - m);
        grad_vec(v[q], j, r.token, scale, c);
        store_vec(r.dx, j, a.V, r.dx_vec, v[q]);
    }
}

int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

// A pair in one cluster (one launch) or all rows, then all pairs, then all rows again (three).
bool pairs_in_clusters(const TokenDesc& d) {
    if (d.n0 == 0 || d.n1 == 0 || d.n0 > 0x7fffffff / kPairCluster) return false;
    // us, a cluster a pair against three launches, L2 flushed before each.  Few and small pairs save two launches: 3
    // of 2x37x257 11 against 13, 60 of 2x32x250 11 against 17, 16 of 2x64x1000 15 against 17; but 16 of 2x128x1000
    // 25 against 19, 128 of 2x64x250 29 against 25.
    const int64_t passes = (d.n1 + 63) / 64;  // rows of a warp
    if (passes <= 2 && passes * ((d.V + 1023) / 1024) <= 4 && d.n0 * passes <= 148) return true;
    // More pairs, while their clusters fill the card and a warp has one to four rows, gain where a row is two to six
    // steps of a warp's walk of 1024 values, so that loads hide its sums and the second read comes partly from L2:
    // 48 of 2x64x4096 51 against 76, 320 of 2x32x4096 143 against 205, 256 of 2x96x4096 348 against 459, 1000 of
    // 2x64x1500 358 against 426, 64 of 2x32x6000 47 against 61; but 16 of 2x128x2000 41 against 29 (SMs without a
    // CTA), 1000 of 2x24x1025 184 against 143 (warps without a row), 74 of 2x192x2000 139 against 125 (six rows a
    // warp), 148 of 2x48x1025 61 against 51 (short rows), 16 of 2x128x8000 126 against 72, 32 of 2x48x8000 70
    // against 56 (long ones).
    return d.n0 * kPairCluster >= 256 && d.n1 >= 64 && passes <= 4 && d.V > 1280 && d.V <= 6144;
}

// Launch configuration of `blocks` CTAs in clusters.
struct Launcher {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    Launcher(int64_t blocks, int threads, size_t smem, int cluster, cudaStream_t stream) {
        cfg.gridDim = dim3(static_cast<unsigned>(blocks));
        cfg.blockDim = dim3(static_cast<unsigned>(threads));
        cfg.dynamicSmemBytes = smem;
        cfg.stream = stream;
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = cluster > 1 ? 1 : 0;
    }
};

template <int G, int NV>
cudaError_t launch_grad(const TokenArgs& a, int cluster, cudaStream_t stream) {
    constexpr size_t smem = kStages * NV * G * 16;
    // clusters that run at the same time, per device and cluster size (found once: the query
    // costs more than a small launch)
    static std::atomic<int> resident[64][kMaxCluster + 1];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    int n = dev < 64 ? resident[dev][cluster].load() : 0;
    if (n == 0) {
        e = cudaFuncSetAttribute(token_grad_kernel<G, NV>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        if (e != cudaSuccess) return e;
        Launcher probe(cluster, G + 32, smem, cluster, stream);
        if (cluster > 1) {
            e = cudaOccupancyMaxActiveClusters(&n, token_grad_kernel<G, NV>, &probe.cfg);
        } else {
            int per_sm = 0, sms = 0;
            e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, token_grad_kernel<G, NV>, G + 32, smem);
            if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
            n = per_sm * sms;
        }
        if (e != cudaSuccess) return e;
        if (n < 1) return cudaErrorInvalidConfiguration;
        if (dev < 64) resident[dev][cluster] = n;
    }
    const int clusters = static_cast<int>(a.rows < n ? a.rows : n);
    Launcher l(static_cast<int64_t>(clusters) * cluster, G + 32, smem, cluster, stream);
    return cudaLaunchKernelEx(&l.cfg, token_grad_kernel<G, NV>, a, clusters);
}

template <bool GRAD>
cudaError_t launch_row_kernel(const TokenArgs& a, cudaStream_t stream) {
    // vectors of a row at most: all rows start on 16 bytes, or one starts up to 3 values behind it
    const bool aligned = reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && a.ls0 % 4 == 0 && a.ls1 % 4 == 0;
    const int vectors = aligned ? (a.V + 3) / 4 : (a.V + 6) / 4;
    // Values alone: a warp a row while the rows are enough to fill the card with warps (V = 4000:
    // 2.5 TB/s with a CTA a row), a CTA or a cluster a row otherwise.
    if (vectors <= 32 * (GRAD ? 16 : 8) || (!GRAD && vectors <= kWalk && a.rows >= 148 * 16)) {
        const int nv = (vectors + 31) / 32;
        const int64_t blocks = (a.rows + 7) / 8;
        if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
        const dim3 grid(static_cast<unsigned>(blocks));
        if (nv <= 1) token_warp_kernel<1, GRAD><<<grid, 256, 0, stream>>>(a);
        else if (nv <= 2) token_warp_kernel<2, GRAD><<<grid, 256, 0, stream>>>(a);
        else if (nv <= 4) token_warp_kernel<4, GRAD><<<grid, 256, 0, stream>>>(a);
        else if (nv <= 8 || !GRAD) token_warp_kernel<8, GRAD><<<grid, 256, 0, stream>>>(a);
        else token_warp_kernel<GRAD ? 16 : 8, GRAD><<<grid, 256, 0, stream>>>(a);
        return cudaGetLastError();
    }
    // As many CTAs a row as hold it, and more while the rows do not fill the card.  Of 256 threads with up to 9
    // vectors each, for which two CTAs an SM have the shared memory (2^27 values, 9 vectors at most against 8:
    // rows of 36000 167 us on 4 CTAs, 178 on 5; 50001 175 on 6, 182 on 7; 9000 177 on 1, 187 on 2; 66000 183,
    // 231 with 512 threads; rows of 18000 are slower, 178 on 2, 175 on 3), then of 512.
    const bool held = GRAD && vectors <= kMaxCluster * 512 * 8;
    const int G = held && vectors > kMaxCluster * 256 * 9 ? 512 : 256, most = G == 256 ? 9 : 8;
    int cluster = held ? (vectors + G * most - 1) / (G * most) : GRAD ? kMaxCluster : 1;
    while (cluster < kMaxCluster && a.rows * cluster < 296 && cluster * G < vectors) ++cluster;
    if constexpr (GRAD) {
        if (held) {
            if (G == 512) return launch_grad<512, 8>(a, cluster, stream);
            // Rows that 128 threads hold, and enough of them: four small CTAs an SM have more rows under way than
            // two (32768 rows of 2500 107 us against 134, 6000 of 2132 29 against 35; but rows of 4000, at 8 vectors
            // a thread, 180 against 154).
            if (vectors <= 128 * 6 && a.rows >= 4 * 148)
                return vectors <= 128 * 5 ? launch_grad<128, 5>(a, 1, stream) : launch_grad<128, 6>(a, 1, stream);
            // no more vectors a thread than it takes: rows of 40000 are 8 a thread of 5 CTAs (9 left the
            // fifth nearly empty and its ring as large as the others')
            switch ((vectors + cluster * G - 1) / (cluster * G)) {
                case 1: case 2: return launch_grad<256, 2>(a, cluster, stream);
                case 3: return launch_grad<256, 3>(a, cluster, stream);
                case 4: return launch_grad<256, 4>(a, cluster, stream);
                case 5: return launch_grad<256, 5>(a, cluster, stream);
                case 6: return launch_grad<256, 6>(a, cluster, stream);
                case 7: return launch_grad<256, 7>(a, cluster, stream);
                case 8: return launch_grad<256, 8>(a, cluster, stream);
                default: return launch_grad<256, 9>(a, cluster, stream);
            }
        }
    }
    if (a.rows * cluster > 0x7fffffff) return cudaErrorInvalidConfiguration;
    Launcher l(a.rows * cluster, kStream, 0, cluster, stream);
    return cudaLaunchKernelEx(&l.cfg, token_stream_kernel<GRAD>, a);
}

}  // namespace

int64_t token_scratch_bytes(const TokenDesc& d) {
    return d.kind == TK_PREFERENCE ? align256(d.n0 * d.n1 * 12) + align256(d.n0 * 4) : 0;
}

int token_launch_count(const TokenDesc& d) {
    const int rows = d.n0 * d.n1 > 0 ? 1 : 0;
    if (d.kind != TK_PREFERENCE) return rows;
    return pairs_in_clusters(d) ? 1 : rows * (d.grad ? 2 : 1) + (d.n0 > 0 ? 1 : 0);
}

int launch_token(const TokenDesc& d, const void* const* in, float* y, float* dlogits, void* scratch, int* status,
                 void* stream) {
    auto f = [&](int k) { return in[k] ? static_cast<const float*>(in[k]) + d.off[k] : nullptr; };
    TokenArgs a;
    a.logits = f(TI_LOGITS);
    a.ls0 = d.s0[TI_LOGITS];
    a.ls1 = d.s1[TI_LOGITS];
    a.tokens = static_cast<const int*>(in[TI_TOKENS]) + d.off[TI_TOKENS];
    a.ts0 = d.s0[TI_TOKENS];
    a.ts1 = d.s1[TI_TOKENS];
    auto operand = [&](int k) { return RowOperand{f(k), d.s0[k], d.s1[k]}; };
    a.old = operand(TI_OLD);
    a.adv = operand(TI_ADVANTAGE);
    a.ref = operand(TI_REF);
    a.g = operand(TI_GRAD);
    a.y = y;
    a.dlogits = dlogits;
    const bool pref = d.kind == TK_PREFERENCE;
    a.stats = pref ? static_cast<float*>(scratch) : nullptr;
    a.slopes = pref && dlogits ? reinterpret_cast<float*>(static_cast<char*>(scratch) + align256(d.n0 * d.n1 * 12)) : nullptr;
    a.status = status;
    a.rows = d.n0 * d.n1;
    a.n1 = d.n1;
    a.V = static_cast<int>(d.V);
    a.kind = d.kind;
    a.f0 = d.f[0];
    a.f1 = d.f[1];
    a.f2 = d.f[2];
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (pref && pairs_in_clusters(d)) {
        Launcher l(d.n0 * kPairCluster, 256, 0, kPairCluster, st);
        if (d.V <= 512) return static_cast<int>(cudaLaunchKernelEx(&l.cfg, preference_cluster_kernel<4>, a));
        return static_cast<int>(cudaLaunchKernelEx(&l.cfg, preference_cluster_kernel<8>, a));
    }
    if (!pref) return a.rows == 0 ? 0 : static_cast<int>(dlogits ? launch_row_kernel<true>(a, st) : launch_row_kernel<false>(a, st));
    // (rounds of as many pairs as stay in L2 between their two reads were slower: 360 against 257 us for
    // 8 pairs of 2x512x16384, the launches' ends costing more than the reads)
    const int64_t per_row = ((a.V + 6) / 4 + kGradVec * kGrad - 1) / (kGradVec * kGrad);
    if (d.n0 > 0x7fffffff || a.rows * per_row > 0x7fffffff) return static_cast<int>(cudaErrorInvalidConfiguration);
    if (d.n0 == 0) return 0;
    if (a.rows > 0) {
        const cudaError_t e = launch_row_kernel<false>(a, st);
        if (e != cudaSuccess) return static_cast<int>(e);
    }
    preference_pair_kernel<<<static_cast<unsigned>(d.n0), kPair, 0, st>>>(a);
    if (dlogits && a.rows > 0 && per_row == 1 && a.rows >= 148 * 8)
        preference_grad_rows_kernel<<<static_cast<unsigned>((a.rows + 7) / 8), 256, 0, st>>>(a);
    else if (dlogits && a.rows > 0)
        preference_grad_kernel<<<static_cast<unsigned>(a.rows * per_row), kGrad, 0, st>>>(a, static_cast<int>(per_row));
    return static_cast<int>(cudaGetLastError());
}

}  // namespace ttb
