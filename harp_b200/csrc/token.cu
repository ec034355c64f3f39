// Log-probabilities of given tokens (entropy, top alternatives), their gradient, and distillation
// from a teacher's top logits: kernels over [N, V] logits rows, V the vocabulary.
//
// With x = scale * z, m = max x, S = sum exp(x - m):
//   logp = (x_t - m) - ln S,  lse = m + ln S,  H = ln S - (sum e_j (x_j - m)) / S,  e_j = exp(x_j - m)
// one pass over the row gives m, S and sum e_j (x_j - m).  All statistics are f32 whatever the logits' type.  The pass
// costs one exponential, and about five other instructions, per logit against 2 or 4 bytes read: f32 rows run at the
// copy rate, 16-bit rows between it and the latencies of a row's end.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "common.h"
#include "tc_ptx.cuh"

namespace eb200 {

namespace {

namespace cg = cooperative_groups;

constexpr int TT = 256;                     // threads per CTA
constexpr int MAX_CLUSTER = 8;
constexpr int MAX_K = 64;                   // alternatives
constexpr int GROUPS = 64;                  // groups of threads whose maxima bound the k-th largest logit, >= MAX_K
constexpr int CAP = 512;                    // candidates held at a time, >= MAX_CLUSTER * MAX_K
constexpr int MAX_TEACHER = 256;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr float NEG_INF = -INFINITY;
constexpr float HEADROOM = 8.f;             // a reference may lie below a logit by this much, in powers of two

__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <class T> struct Pack { static constexpr int E = 16 / sizeof(T); };   // logits in 16 bytes

__device__ __forceinline__ void unpack(const uint4& u, float (&x)[4], float) {
    x[0] = __uint_as_float(u.x); x[1] = __uint_as_float(u.y); x[2] = __uint_as_float(u.z); x[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void unpack(const uint4& u, float (&x)[8], __nv_bfloat16) {
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
__device__ __forceinline__ void unpack(const uint4& u, float (&x)[8], __half) {
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x; x[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ uint4 pack(const float (&x)[4], float) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
}
__device__ __forceinline__ uint4 pack(const float (&x)[8], __nv_bfloat16) {
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) { const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]); w[i] = *reinterpret_cast<const unsigned*>(&h); }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 pack(const float (&x)[8], __half) {
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) { const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]); w[i] = *reinterpret_cast<const unsigned*>(&h); }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ long long load_id(const void* ids, long long i, bool wide) {
    return wide ? __ldg(reinterpret_cast<const long long*>(ids) + i) : (long long)__ldg(reinterpret_cast<const int*>(ids) + i);
}

// A row in slots of 16 aligned bytes: slot s holds logits s * E - lead + [0, E).  The first and the last
// slot may reach over the row's ends; nothing outside the row is ever read.
template <class T> struct Row {
    static constexpr int E = Pack<T>::E;
    const T* p;
    int v, lead, slots;
    __device__ Row(const T* row, int v_) : p(row), v(v_) {
        lead = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
        slots = (lead + v + E - 1) / E;
    }
    __device__ bool whole(int s) const { return s * E >= lead && (s + 1) * E <= lead + v; }
    __device__ uint4 raw(int s) const { return __ldg(reinterpret_cast<const uint4*>(p - lead) + s); }
    __device__ void part(int s, float (&x)[E]) const {
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int j = s * E - lead + i;
            x[i] = j >= 0 && j < v ? to_f(__ldg(p + j)) : NEG_INF;
        }
    }
};

// ---- row statistics --------------------------------------------------------------------------------

// A thread's sums are held against a reference 2^rc of its own, rc a whole number, so that moving or joining
// references scales by powers of two: s = sum e, t = sum e * y over y = x * c - rc (one rounding), e = 2^y,
// c = scale * log2(e).  rc is set by the first logits and moves when y would exceed HEADROOM.  mx is the largest
// logit seen, slot the first slot that holds it (-1: no slot seen).  Logits below -FAR / c (masks) never set a
// reference and count as 0; a row whose maximum lies beyond NEAR / c is summed again against that maximum.
constexpr float NEAR = 4194304.f, FAR = 8388608.f;

typedef unsigned long long f32x2;

struct Acc {
    float rc = 0.f, lim, mx = NEG_INF;
    f32x2 s = 0, t = 0;                                   // two sums each, of even and odd places
    int slot = -1;
    __device__ __forceinline__ explicit Acc(float c) : lim(-FAR / c) {}
};

// y of a logit far below its reference counts as -1000: e is 0 there and e * y must not be 0 * inf
__device__ __forceinline__ float floor_y(float y) { return fmaxf(y, -1000.f); }

// two f32 in a 64-bit register
__device__ __forceinline__ f32x2 pair(float lo, float hi) { f32x2 d; asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi)); return d; }
__device__ __forceinline__ float2 parts(f32x2 a) { float2 d; asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(a)); return d; }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) { f32x2 d; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c)); return d; }
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) { f32x2 d; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b)); return d; }

__device__ __forceinline__ void move_reference(Acc& a, float mx, float c) {
    const float rc = fminf(rintf(mx * c), FAR);
    const float dy = fminf(floor_y(a.rc - rc), 0.f), f = ex2(dy);       // 0 sums before the first reference
    const f32x2 ff = pair(f, f);
    a.t = fma2(ff, fma2(pair(dy, dy), a.s, a.t), 0);
    a.s = fma2(ff, a.s, 0);
    a.rc = rc;
    a.lim = (rc + HEADROOM) / c;
}

// 16 bytes of logits as they lie in memory: their maximum (NaN left out), and pairs of them in f32.  With an entropy,
// -inf becomes a finite value whose e is 0 (`low`; NaN stays).
template <class T> struct Bits;
template <> struct Bits<float> {
    static __device__ __forceinline__ unsigned more(unsigned a, unsigned b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }
    static __device__ __forceinline__ uint4 larger(const uint4& a, const uint4& b) { return make_uint4(more(a.x, b.x), more(a.y, b.y), more(a.z, b.z), more(a.w, b.w)); }
    static __device__ __forceinline__ float largest(const uint4& u) {
        return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
    }
    template <bool ENT> static __device__ __forceinline__ void pairs(const uint4& u, float2 (&x)[2], float c) {
        x[0] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
        x[1] = make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
        if (ENT) {
            const float low = fmaxf(-2.f * FAR / c, -3.402823466e38f);
#pragma unroll
            for (int i = 0; i < 2; ++i) { x[i].x = x[i].x < low ? low : x[i].x; x[i].y = x[i].y < low ? low : x[i].y; }
        }
    }
};
template <> struct Bits<__nv_bfloat16> {
    static __device__ __forceinline__ __nv_bfloat162 as(unsigned w) { return *reinterpret_cast<__nv_bfloat162*>(&w); }
    static __device__ __forceinline__ unsigned more(unsigned a, unsigned b) { const __nv_bfloat162 m = __hmax2(as(a), as(b)); return *reinterpret_cast<const unsigned*>(&m); }
    static __device__ __forceinline__ uint4 larger(const uint4& a, const uint4& b) { return make_uint4(more(a.x, b.x), more(a.y, b.y), more(a.z, b.z), more(a.w, b.w)); }
    static __device__ __forceinline__ float largest(const uint4& u) {
        const __nv_bfloat162 m = __hmax2(__hmax2(as(u.x), as(u.y)), __hmax2(as(u.z), as(u.w)));
        return fmaxf(__low2float(m), __high2float(m));
    }
    template <bool ENT> static __device__ __forceinline__ void pairs(const uint4& u, float2 (&x)[4], float c) {
        unsigned w[4] = {u.x, u.y, u.z, u.w};
        const __nv_bfloat162 low = __float2bfloat162_rn(fmaxf(-2.f * FAR / c, -3.3e38f));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (ENT) { const __nv_bfloat162 h = __hmax2_nan(as(w[i]), low); w[i] = *reinterpret_cast<const unsigned*>(&h); }
            x[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
        }
    }
};
template <> struct Bits<__half> {
    static __device__ __forceinline__ __half2 as(unsigned w) { return *reinterpret_cast<__half2*>(&w); }
    static __device__ __forceinline__ unsigned more(unsigned a, unsigned b) { const __half2 m = __hmax2(as(a), as(b)); return *reinterpret_cast<const unsigned*>(&m); }
    static __device__ __forceinline__ uint4 larger(const uint4& a, const uint4& b) { return make_uint4(more(a.x, b.x), more(a.y, b.y), more(a.z, b.z), more(a.w, b.w)); }
    static __device__ __forceinline__ float largest(const uint4& u) {
        const __half2 m = __hmax2(__hmax2(as(u.x), as(u.y)), __hmax2(as(u.z), as(u.w)));
        return fmaxf(__low2float(m), __high2float(m));
    }
    template <bool ENT> static __device__ __forceinline__ void pairs(const uint4& u, float2 (&x)[4], float) {
        const unsigned w[4] = {u.x, u.y, u.z, u.w};
        const __half2 low = __float2half2_rn(-65504.f);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __half22float2(ENT ? __hmax2_nan(as(w[i]), low) : as(w[i]));
    }
};

template <bool ENT>
__device__ __forceinline__ void add_pair(Acc& a, float2 x, f32x2 c, f32x2 minus_rc) {
    const f32x2 y = fma2(pair(x.x, x.y), c, minus_rc);
    const float2 p = parts(y);
    const f32x2 e = pair(ex2(p.x), ex2(p.y));
    a.s = add2(a.s, e);
    if (ENT) a.t = fma2(e, y, a.t);
}

// N slots of a thread: one comparison against the reference for all of them
template <class T, bool ENT, bool TOP, int N>
__device__ __forceinline__ void take(Acc& a, const uint4 (&u)[N], int slot, int step, float c) {
    float mx = NEG_INF;
    if (TOP) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float m = Bits<T>::largest(u[i]);
            if (m > a.mx) { a.mx = m; a.slot = slot + i * step; }
            mx = fmaxf(mx, m);
        }
    } else {
        uint4 m = u[0];
#pragma unroll
        for (int i = 1; i < N; ++i) m = Bits<T>::larger(m, u[i]);
        mx = fmaxf(mx, Bits<T>::largest(m));
        a.mx = fmaxf(a.mx, mx);
    }
    if (mx > a.lim) move_reference(a, mx, c);
    const f32x2 cc = pair(c, c), minus_rc = pair(-a.rc, -a.rc);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float2 x[Pack<T>::E / 2];
        Bits<T>::template pairs<ENT>(u[i], x, c);
#pragma unroll
        for (int q = 0; q < Pack<T>::E / 2; ++q) add_pair<ENT>(a, x[q], cc, minus_rc);
    }
}

// a slot that reaches over the row's ends (its places outside hold -inf)
template <class T, bool ENT, bool TOP>
__device__ __forceinline__ void take_part(Acc& a, const float (&x)[Pack<T>::E], int slot, float c) {
    float mx = NEG_INF;
#pragma unroll
    for (int i = 0; i < Pack<T>::E; ++i) mx = fmaxf(mx, x[i]);
    if (TOP && (mx > a.mx || (mx == a.mx && slot < a.slot))) a.slot = slot;      // the row's first slot is taken last
    a.mx = fmaxf(a.mx, mx);
    if (mx > a.lim) move_reference(a, mx, c);
#pragma unroll
    for (int i = 0; i < Pack<T>::E; ++i) {
        const float y = fmaf(x[i], c, -a.rc), e = ex2(y);
        a.s = add2(a.s, pair(e, 0.f));
        if (ENT) a.t = add2(a.t, pair(e * floor_y(y), 0.f));
    }
}

struct Stat { float rc, s, t, mx; };

__device__ __forceinline__ Stat join(const Stat& a, const Stat& b) {
    Stat o;
    o.rc = fmaxf(a.rc, b.rc);
    const float da = floor_y(a.rc - o.rc), db = floor_y(b.rc - o.rc), fa = ex2(da), fb = ex2(db);
    o.s = fa * a.s + fb * b.s;
    o.t = fa * fmaf(da, a.s, a.t) + fb * fmaf(db, b.s, b.t);
    o.mx = fmaxf(a.mx, b.mx);
    return o;
}

template <int CT> struct StatShared { Stat warp[CT / 32], cta[MAX_CLUSTER]; };

// the barrier of the CT threads that take logits
template <int CT> __device__ __forceinline__ void rows_sync() { asm volatile("bar.sync 1, %0;" ::"n"(CT) : "memory"); }

// the CTA's totals on all those threads, joined in the same order everywhere
template <int CT>
__device__ __forceinline__ Stat cta_totals(const Acc& a, StatShared<CT>& sh) {
    const float2 sp = parts(a.s), tp = parts(a.t);
    const float s = sp.x + sp.y;
    Stat st = {s == 0.f ? -2.f * FAR : a.rc, s, tp.x + tp.y, a.mx};
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
        Stat q;
        q.rc = __shfl_xor_sync(~0u, st.rc, o); q.s = __shfl_xor_sync(~0u, st.s, o);
        q.t = __shfl_xor_sync(~0u, st.t, o); q.mx = __shfl_xor_sync(~0u, st.mx, o);
        st = join(st, q);
    }
    if ((threadIdx.x & 31) == 0) sh.warp[threadIdx.x >> 5] = st;
    rows_sync<CT>();
    st = sh.warp[0];
#pragma unroll
    for (int w = 1; w < CT / 32; ++w) st = join(st, sh.warp[w]);
    return st;
}

// The CTAs of a cluster hand each other their totals (and CTA 0 their alternatives): plain stores into the peer's
// shared memory, then an arrival at the peer's mbarrier.  Every CTA waits for all the others' before it ends, so no
// store reaches a CTA that has gone.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ void arrive_at(uint64_t* bar, int cta) {
    asm volatile("{ .reg .b32 a; mapa.shared::cluster.u32 a, %0, %1; mbarrier.arrive.release.cluster.shared::cluster.b64 _, [a]; }"
                 ::"r"(smem_u32(bar)), "r"(cta) : "memory");
}
__device__ __forceinline__ void wait_cluster(uint64_t* bar, int* error_flag) {
    for (unsigned i = 0; i < TC_SPIN_LIMIT; ++i) {
        unsigned ok;
        asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], 0; selp.u32 %0, 1, 0, p; }"
                     : "=r"(ok) : "r"(smem_u32(bar)) : "memory");
        if (ok) return;
        if (i > 4096) __nanosleep(64);
    }
    atomicExch(error_flag, 1);
}

template <int CT>
__device__ __forceinline__ Stat exchange(const Stat& mine, StatShared<CT>& sh, uint64_t* bar, int cluster, int rank, int* error_flag) {
    const int tid = threadIdx.x;
    if (tid < cluster) cg::this_cluster().map_shared_rank(&sh, tid)->cta[rank] = mine;
    rows_sync<CT>();                        // all stores of this CTA lie before its arrivals
    if (tid < cluster) arrive_at(bar, tid);
    wait_cluster(bar, error_flag);
    Stat st = sh.cta[0];
    for (int i = 1; i < cluster; ++i) st = join(st, sh.cta[i]);
    return st;
}

// against the row's maximum m: S >= 1, ln S >= 0, and mean = sum e (x - m) / S <= 0.  A row of -inf is `empty`.
struct Final { float m, s, ln_s, mean; bool empty; };

// The largest logit's own terms, rounded here as they were when they were added, come off both sums first: what the
// others leave is 0 for a row of one possible logit, so its ln S and its entropy are exactly 0, and no rounding can make
// a probability larger than 1 or an entropy negative.  (s * 2^-dy, two roundings, gave S < 1 on every fifth such row.)
__device__ __forceinline__ Final finish(const Stat& st, float c) {
    Final f;
    f.m = st.mx;
    f.empty = st.mx == NEG_INF && st.s == 0.f;                  // a NaN makes s NaN
    if (f.empty) { f.s = 1.f; f.ln_s = 0.f; f.mean = 0.f; return f; }
    const float dy = fmaf(st.mx, c, -st.rc), own = ex2(dy), rest = st.s - own;
    float others = rest * ex2(-dy), mean = LN2 * (fmaf(-dy, rest, st.t - __fmul_rn(own, dy)) / st.s);
    if (others < 0.f) others = 0.f;                             // NaN stays
    if (mean > 0.f) mean = 0.f;
    f.s = 1.f + others;
    f.ln_s = logf(f.s);                                         // of `others` no digits are left that log1p would keep
    f.mean = mean;
    return f;
}

// Rows that are summed again against their maximum: beyond NEAR (logits of millions, or nothing but a mask's lowest
// value), +inf, or -- with an entropy -- f16 whose maximum is so near -65504 (what -inf became) that this would count.
template <class T, bool ENT> __device__ __forceinline__ bool again(float m, float c) {
    const bool low_range = ENT && std::is_same<T, __half>::value && c * (m + 65504.f) < 400.f;
    return m != NEG_INF && (fabsf(m) * c >= NEAR || low_range);
}

template <bool ENT, int E> __device__ __forceinline__ void take_against(Acc& b, const float (&x)[E], float m, float c) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const float y = (x[i] - m) * c, e = ex2(y);
        b.s = add2(b.s, pair(e, 0.f));
        if (ENT) b.t = add2(b.t, pair(e * floor_y(y), 0.f));
    }
}
__device__ __forceinline__ Final finish_against(const Stat& st, float m) { return {m, st.s, logf(st.s), LN2 * (st.t / st.s), false}; }

// ---- top alternatives ------------------------------------------------------------------------------
// Order of a logit as an unsigned whole number (NaN like -inf, -0 like 0); 0 is below every logit.
__device__ __forceinline__ unsigned order_of(float x) {
    if (x != x) x = NEG_INF;
    const unsigned b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
// larger value first, then lower index: unique per logit of a row
__device__ __forceinline__ unsigned long long key_of(unsigned order, unsigned index) { return (unsigned long long)order << 32 | (0xffffffffu - index); }
__device__ __forceinline__ unsigned index_of(unsigned long long key) { return 0xffffffffu - (unsigned)key; }

struct TopShared {
    unsigned long long keys[TT], groups[GROUPS], cand[CAP], peers[MAX_CLUSTER * MAX_K];
    unsigned long long tau;
    int owners[TT];
    int n_owners, n_cand, n_peers[MAX_CLUSTER];
};

// keeps the k largest of cand[0, n), sorted; all threads; returns how many there are
__device__ __forceinline__ int keep_largest(TopShared& sh, int n, int k) {
    constexpr int PER = CAP / TT;
    unsigned long long mine[PER];
    int rank[PER];
    rows_sync<TT>();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int at = threadIdx.x + i * TT;
        rank[i] = CAP;
        if (at < n) {
            mine[i] = sh.cand[at];
            int r = 0;
            for (int j = 0; j < n; ++j) r += sh.cand[j] > mine[i];
            rank[i] = r;
        }
    }
    rows_sync<TT>();
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (rank[i] < k) sh.cand[rank[i]] = mine[i];
    rows_sync<TT>();
    return min(n, k);
}

// The k largest logits of this CTA's slots (first + tid + i * step) into sh.cand, sorted; returns how many.
// The k-th largest of 64 group maxima bounds the k-th largest logit from below, so only threads whose
// maximum reaches it hold candidates; their slots (about 1.3 k threads' worth) are read again, by all threads.
// get(s, x) brings slot s < end.
template <class T, class GET>
__device__ __forceinline__ int top_of_cta(TopShared& sh, const Acc& a, const Row<T>& row, int first, int step, int end, int k, GET get) {
    constexpr int E = Pack<T>::E;
    const int tid = threadIdx.x;
    const unsigned long long key = a.slot < 0 ? 0 : key_of(order_of(a.mx), a.slot);
    sh.keys[tid] = key;
    if (tid == 0) sh.n_owners = sh.n_cand = 0;
    rows_sync<TT>();
    if (tid < GROUPS) {
        unsigned long long g = 0;
#pragma unroll
        for (int i = 0; i < TT / GROUPS; ++i) g = max(g, sh.keys[tid + i * GROUPS]);
        sh.groups[tid] = g;
    }
    rows_sync<TT>();
    if (tid < GROUPS) {
        const unsigned long long g = sh.groups[tid];
        int r = 0;
#pragma unroll 8
        for (int j = 0; j < GROUPS; ++j) r += sh.groups[j] > g || (sh.groups[j] == g && j < tid);
        if (r == k - 1) sh.tau = g;
    }
    rows_sync<TT>();
    const unsigned long long tau = sh.tau;
    const unsigned tau_order = (unsigned)(tau >> 32);
    const int tau_slot = (int)(0xffffffffu - (unsigned)tau);       // equal values count up to the end of this slot
    if (key != 0 && key >= tau) sh.owners[atomicAdd(&sh.n_owners, 1)] = tid;
    rows_sync<TT>();
    const int n_own = sh.n_owners, per = (end - first + step - 1) / step;
    const long long pairs = (long long)n_own * per;
    auto collect = [&](long long pair) {
        const int s = first + sh.owners[(int)(pair % n_own)] + (int)(pair / n_own) * step;
        if (s >= end) return;
        float x[E];
        get(s, x);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const unsigned o = order_of(x[i]);
            const int j = s * E - row.lead + i;
            if (j >= 0 && j < row.v && (tau == 0 || o > tau_order || (o == tau_order && s <= tau_slot))) {
                const int at = atomicAdd(&sh.n_cand, 1);
                if (at < CAP) sh.cand[at] = key_of(o, j);
            }
        }
    };
    for (long long p = tid; p < pairs; p += TT) collect(p);
    rows_sync<TT>();
    int n = sh.n_cand;
    if (n > CAP) {
        // more than fit (large logits gathered in a few threads' slots): some slots at a time, keeping the k largest
        constexpr int CHUNK = (CAP - MAX_K) / E / 32 * 32;
        n = 0;
        for (long long p0 = 0; p0 < pairs; p0 += CHUNK) {
            rows_sync<TT>();
            if (tid == 0) sh.n_cand = n;
            rows_sync<TT>();
            const long long p1 = min(p0 + CHUNK, pairs);
            for (long long p = p0 + tid; p < p1; p += TT) collect(p);
            rows_sync<TT>();
            n = keep_largest(sh, sh.n_cand, k);
        }
        return n;
    }
    return keep_largest(sh, n, k);
}

// The CTAs' candidates at CTA 0 of the cluster: sent, and after a cluster barrier merged there.
__device__ __forceinline__ void send_top(TopShared& sh, int have, int rank) {
    TopShared* lead = cg::this_cluster().map_shared_rank(&sh, 0);
    if ((int)threadIdx.x < have) lead->peers[rank * MAX_K + threadIdx.x] = sh.cand[threadIdx.x];
    if (threadIdx.x == 0) lead->n_peers[rank] = have;
}
__device__ __forceinline__ void merge_top(TopShared& sh, int cluster, int k) {
    if (threadIdx.x == 0) sh.n_cand = 0;
    rows_sync<TT>();
    for (int i = threadIdx.x; i < cluster * MAX_K; i += TT)
        if (i % MAX_K < sh.n_peers[i / MAX_K]) sh.cand[atomicAdd(&sh.n_cand, 1)] = sh.peers[i];
    rows_sync<TT>();
    keep_largest(sh, sh.n_cand, k);
}

// ---- forward ---------------------------------------------------------------------------------------

struct LogprobOut { float *logp, *lse, *entropy, *top; int* top_ids; };

// ---- 16 bytes of logits from any element address ---------------------------------------------------

// bytes [shift, shift + 16) of the 32 bytes (a, b)
__device__ __forceinline__ uint4 shifted(const uint4& a, const uint4& b, int shift) {
    const unsigned bits = (shift & 3) * 8;
    unsigned w[5];
    switch (shift >> 2) {
        case 0: w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = b.x; break;
        case 1: w[0] = a.y; w[1] = a.z; w[2] = a.w; w[3] = b.x; w[4] = b.y; break;
        case 2: w[0] = a.z; w[1] = a.w; w[2] = b.x; w[3] = b.y; w[4] = b.z; break;
        default: w[0] = a.w; w[1] = b.x; w[2] = b.y; w[3] = b.z; w[4] = b.w; break;
    }
    return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits), __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
}

// logits [j, j + E) of a row of v that starts at p, element by element where the 16 aligned bytes around them (two times
// 16 if `shift`, the bytes by which p + j lies beyond a boundary) leave the row
template <class T> __device__ __forceinline__ void window(const T* p, int v, int j, int shift, float (&x)[Pack<T>::E]) {
    constexpr int E = Pack<T>::E;
    const int down = shift / (int)sizeof(T);
    const uint4* at = reinterpret_cast<const uint4*>(p + j - down);
    if (shift == 0 && j >= 0 && j + E <= v) unpack(__ldg(at), x, T());
    else if (shift != 0 && j - down >= 0 && j - down + 2 * E <= v) unpack(shifted(__ldg(at), __ldg(at + 1), shift), x, T());
    else {
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = j + i >= 0 && j + i < v ? to_f(__ldg(p + j + i)) : NEG_INF;
    }
}

template <class T> __device__ __forceinline__ void put(T* p, int v, int j, const float (&y)[Pack<T>::E]) {
    constexpr int E = Pack<T>::E;
    if (j >= 0 && j + E <= v) {
        *reinterpret_cast<uint4*>(p + j) = pack(y, T());
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (j + i >= 0 && j + i < v) p[j + i] = from_f<T>(y[i]);
    }
}

// ---- gradient --------------------------------------------------------------------------------------
// d_j = scale * (g_l ([j = t] - p_j) - g_H p_j (ln p_j + H)), p_j = exp(x_j - lse): a stream of logits in and a
// stream of gradients out, cut along 16-byte slots of the output so that stores stay whole whatever the pitches.
// A CTA takes GU * 256 slots of a row; all of them whole is the rule, and then nothing is tested per slot.  DRAM bounds
// it: 4096 x 131072 bf16 with the entropy's term takes 344 us back to back, 362 among other work (6.2 and 5.9 TB/s; a warp
// per 128 slots with tests per slot: 513).  Rows out of step with their output load every slot twice and shift: 1023 x
// 50021 f16 takes 43 us, 4.7 TB/s.
constexpr int GU = 4;

// lse in f32 is off by up to a quarter from here on (rows of a mask's lowest value, logits of millions): x_j - lse may then
// round far above 0, and is held at 0, so that p_j stays a probability.  Below, p_j is off by what lse's rounding makes it.
constexpr float FAR_LSE = 4194304.f;

struct GradArgs {
    const void* z;
    void* g;
    long long pitch, g_pitch, rows;
    int v, per_row;
    float scale;
    const void* ids;
    int wide;
    const float *lse, *g_logp, *entropy, *g_entropy;
};

template <class T, bool ENT>
__global__ void __launch_bounds__(TT, 5) token_logprob_grad_kernel(const GradArgs a) {
    constexpr int E = Pack<T>::E;
    const int v = a.v, tid = threadIdx.x;
    const long long n = blockIdx.x / a.per_row;
    const int s0 = (int)(blockIdx.x % a.per_row) * GU * TT + tid;
    const T* p = reinterpret_cast<const T*>(a.z) + n * a.pitch;
    T* o = reinterpret_cast<T*>(a.g) + n * a.g_pitch;
    const long long t = load_id(a.ids, n, a.wide);
    const float norm = __ldg(a.lse + n), gl = t >= 0 && t < v ? __ldg(a.g_logp + n) : 0.f;
    const float gh = ENT ? __ldg(a.g_entropy + n) : 0.f, h = ENT ? __ldg(a.entropy + n) : 0.f;
    const int lead = (int)((reinterpret_cast<uintptr_t>(o) & 15) / sizeof(T));
    const int slots = (lead + v + E - 1) / E;
    const int shift = (int)(reinterpret_cast<uintptr_t>(p - lead) & 15);
    const bool zero = norm == NEG_INF || (gl == 0.f && gh == 0.f), far = fabsf(norm) >= FAR_LSE;
    const float up = gl * a.scale, ah = -gh * a.scale;

    auto gradient = [&](float (&x)[E], int s, bool hold) {
#pragma unroll
        for (int q = 0; q < E; ++q) {
            float d = fmaf(x[q], a.scale, -norm);
            if (hold && d > 0.f) d = 0.f;
            const float pr = ex2(d * LOG2E);
            x[q] = pr * (ENT ? fmaf(ah, floor_y(d) + h, -up) : -up);
        }
        const long long at = t - ((long long)s * E - lead);
        if (at >= 0 && at < E) {
#pragma unroll
            for (int q = 0; q < E; ++q) x[q] += q == (int)at ? up : 0.f;
        }
    };

    const int lo = s0 - tid, hi = lo + GU * TT;
    if (!zero && !far && lo * E - lead - (shift ? E : 0) >= 0 && (hi + (shift ? 1 : 0)) * E - lead <= v) {
        const uint4* from = reinterpret_cast<const uint4*>(p - lead - shift / (int)sizeof(T)) + s0;
        uint4* to = reinterpret_cast<uint4*>(o - lead) + s0;
        uint4 u[GU];
        if (shift == 0) {
#pragma unroll
            for (int i = 0; i < GU; ++i) u[i] = __ldcs(from + i * TT);
        } else {
            uint4 w[GU];
#pragma unroll
            for (int i = 0; i < GU; ++i) { u[i] = __ldg(from + i * TT); w[i] = __ldg(from + i * TT + 1); }
#pragma unroll
            for (int i = 0; i < GU; ++i) u[i] = shifted(u[i], w[i], shift);
        }
#pragma unroll
        for (int i = 0; i < GU; ++i) {
            float x[E];
            unpack(u[i], x, T());
            gradient(x, s0 + i * TT, false);
            __stcs(to + i * TT, pack(x, T()));
        }
        return;
    }
    for (int s = s0; s < min(hi, slots); s += TT) {
        const int j = s * E - lead;
        float x[E];
        if (zero) {
#pragma unroll
            for (int q = 0; q < E; ++q) x[q] = 0.f;
        } else {
            window(p, v, j, shift, x);
            gradient(x, s, far);
        }
        put(o, v, j, x);
    }
}

// ---- distillation ----------------------------------------------------------------------------------
// L = sum_k q_k (ln q_k - ln p_{c_k}), q = softmax of the teacher's K values; dL/dz_j = scale * (p_j - sum_{c_k = j} q_k).
// Warp 0 forms q while the other warps are on the row.  The gradient is the dense scale * weight * p_j first; after a
// barrier the teacher's places are written again with their q taken off, each from f32 and rounded once.
struct Teacher {
    const void *values, *ids;
    int dtype, wide;
    __device__ __forceinline__ float value(long long i) const {
        if (dtype == EB200_F32) return __ldg(reinterpret_cast<const float*>(values) + i);
        if (dtype == EB200_F16) return to_f(__ldg(reinterpret_cast<const __half*>(values) + i));
        return to_f(__ldg(reinterpret_cast<const __nv_bfloat16*>(values) + i));
    }
};

struct TeacherShared {
    float q[MAX_TEACHER], ln_q[MAX_TEACHER], z[MAX_TEACHER];
    int id[MAX_TEACHER];
    int some;
};

template <class T>
__device__ __forceinline__ void teacher_row(TeacherShared& sh, const T* p, int v, const Teacher& te, long long n, int k, float c) {
    constexpr int PER = MAX_TEACHER / 32;
    const int lane = threadIdx.x & 31;
    float u[PER], mx = NEG_INF;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int at = lane + i * 32;
        u[i] = NEG_INF;
        if (at < k) {
            const long long id = load_id(te.ids, n * k + at, te.wide);
            const bool there = id >= 0 && id < v;
            if (there) u[i] = te.value(n * k + at);
            sh.id[at] = there ? (int)id : -1;
            sh.z[at] = there ? to_f(__ldg(p + id)) : NEG_INF;
        }
        mx = fmaxf(mx, u[i]);
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, o));
    const float r = mx == NEG_INF ? 0.f : mx;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) { u[i] = (u[i] - r) * c; s += ex2(u[i]); }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    const float ln_s = logf(s);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int at = lane + i * 32;
        if (at < k) {
            sh.q[at] = s == 0.f ? 0.f : ex2(u[i]) / s;
            sh.ln_q[at] = u[i] * LN2 - ln_s;
        }
    }
    if (lane == 0) sh.some = s != 0.f;        // NaN counts
}

// by one warp
__device__ __forceinline__ float distill_loss(const TeacherShared& sh, const Final& f, int k, float scale) {
    float l = 0.f;
    for (int i = threadIdx.x & 31; i < k; i += 32) {
        const float q = sh.q[i], lp = f.empty ? NEG_INF : (sh.z[i] - f.m) * scale - f.ln_s;
        if (!(q == 0.f)) l += q * (sh.ln_q[i] - lp);
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) l += __shfl_xor_sync(~0u, l, o);
    return l;
}

// ---- longer rows -----------------------------------------------------------------------------------
// CTAs that stay take rows in turn.  One thread keeps a ring of chunks in shared memory filled by bulk copies, running
// ahead into the next row while this one is being finished, so what is in flight depends neither on registers nor on
// where a row ends; one warp fetches what else a row needs (the token's logit, the teacher's entries), a row ahead;
// CT threads take the logits.  Few rows: the CTAs of a cluster share one, each a slice of whole slots.
// The distillation gradient has the row's chunks brought a second time.  L2 serves that while the rows in work (one CTA
// per SM, 148 rows) and the gradient written meanwhile fit: 1024 x 131072 bf16 reads 275 MB of DRAM, one reading; at 512 KB
// a row (f32) it reads 926 MB, so most second readings miss.  4096 x 131072: bf16 445 to 477 us (1.3 to 1.4 times its
// bytes at the copy rate; with four CTAs per SM, whose second reading missed, 620), f32 997 us (1.5 times).
// The forward pass of 4096 x 131072 takes 330 us in f32 (6.5 TB/s), 184 to 215 in bf16 (reading 1.07 GB at the copy rate
// would take 166): the exponentials' unit works in 68 % of an SM's active cycles and 57 % of all, the rest is latency at
// rows' ends and the tenth turn of 4096 rows on 444 CTAs.  Two and four CTAs per SM came within 3 % of three.
enum { ROWS_LOGPROB, ROWS_TOP, ROWS_DISTILL, ROWS_DISTILL_GRAD };

struct RowsArgs {
    const void* z;
    long long pitch, rows;
    int v, k;
    float scale;
    const void* ids;
    int wide;
    LogprobOut out;
    Teacher te;
    const float* weights;
    float* loss;
    void* g;
    long long g_pitch;
    int cluster, per;                       // slots per CTA of a row
    int* error_flag;
};

template <int MODE> struct RowsShape {
    static constexpr int CT = MODE == ROWS_DISTILL_GRAD ? 512 : TT;       // threads that take logits
    static constexpr int CTAS = MODE == ROWS_DISTILL_GRAD ? 1 : 3;        // per SM
    static constexpr int CHUNK = 4 * CT;                                  // slots per copy: 16 or 32 KB
    static constexpr int STAGES = MODE == ROWS_DISTILL_GRAD ? 6 : MODE == ROWS_TOP ? 3 : 4;
    static constexpr int STAGE_BYTES = CHUNK * 16 + (MODE == ROWS_DISTILL_GRAD ? 128 : 0);      // one more slot for windows over the chunk's end
    static constexpr int THREADS = CT + 64;                               // and the copying thread's warp, and the fetching one
};

struct OwnLogit { float z; int there; };
struct Edges { uint4 head, tail; };          // the row's slots that reach over its ends

template <int MODE> struct RowsShared {
    using S = RowsShape<MODE>;
    unsigned char ring[S::STAGES][S::STAGE_BYTES];
    uint64_t full[S::STAGES], empty[S::STAGES], side_full[2], side_empty[2], peers[2];
    alignas(16) StatShared<S::CT> stat[2], second;
    Edges edges[2];
    OwnLogit own[2];
    float weight[2];
    TeacherShared teach[MODE >= ROWS_DISTILL ? 2 : 1];
};
template <> struct RowsShared<ROWS_TOP> {
    using S = RowsShape<ROWS_TOP>;
    unsigned char ring[S::STAGES][S::STAGE_BYTES];
    uint64_t full[S::STAGES], empty[S::STAGES], side_full[2], side_empty[2], peers[2];
    alignas(16) StatShared<S::CT> stat[2], second;
    Edges edges[2];
    OwnLogit own[2];
    TopShared top;
};

// the whole slots [w0, w1) among the m slots of this CTA's slice, which begins at slot `first`
struct Slice {
    int first, m, w0, w1;
    __device__ bool tail() const { return w1 < m && m - 1 >= w0; }
};
template <class T> __device__ __forceinline__ Slice slice_of(const Row<T>& row, int rank, int per) {
    Slice s;
    s.first = rank * per;
    s.m = max(0, min(row.slots - s.first, per));
    s.w0 = s.m > 0 && !row.whole(s.first) ? 1 : 0;
    s.w1 = s.m > 0 && !row.whole(s.first + s.m - 1) ? max(s.m - 1, s.w0) : s.m;
    return s;
}

template <class T, int MODE>
__global__ void __launch_bounds__(RowsShape<MODE>::THREADS, RowsShape<MODE>::CTAS) token_rows_kernel(const RowsArgs a) {
    using S = RowsShape<MODE>;
    constexpr int E = Pack<T>::E, CT = S::CT, CHUNK = S::CHUNK, STAGES = S::STAGES, U = CHUNK / CT;
    constexpr bool TOP = MODE == ROWS_TOP, ENT = MODE <= ROWS_TOP, DISTILL = MODE >= ROWS_DISTILL, GRAD = MODE == ROWS_DISTILL_GRAD;
    extern __shared__ __align__(128) unsigned char dyn[];
    RowsShared<MODE>& sh = *reinterpret_cast<RowsShared<MODE>*>(dyn);
    const int tid = threadIdx.x, warp = tid >> 5, cluster = a.cluster, rank = blockIdx.x % cluster;
    const long long n0 = blockIdx.x / cluster, step = gridDim.x / cluster;
    const float c = a.scale * LOG2E;

    if (tid == 0) {
        for (int i = 0; i < STAGES; ++i) { mbar_init(&sh.full[i], 1); mbar_init(&sh.empty[i], CT / 32); }
        for (int i = 0; i < 2; ++i) { mbar_init(&sh.side_full[i], 1); mbar_init(&sh.side_empty[i], CT / 32); mbar_init(&sh.peers[i], cluster); }
        asm volatile("fence.mbarrier_init.release.cluster; fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    if (cluster > 1) cluster_arrive();      // waited for before the first store into another CTA

    if (warp == CT / 32) {                  // ---- copies ----
        if ((tid & 31) == 0) {
            unsigned it = 0;
            for (long long n = n0; n < a.rows; n += step) {
                const Row<T> row(reinterpret_cast<const T*>(a.z) + n * a.pitch, a.v);
                const Slice sl = slice_of(row, rank, a.per);
                const uint4* src = reinterpret_cast<const uint4*>(row.p - row.lead) + sl.first;
                for (int round = 0; round < (GRAD ? 2 : 1); ++round) {
                    for (int lo = 0; lo < sl.w1; lo += CHUNK, ++it) {
                        const int st = it % STAGES, b = max(lo, sl.w0), e = min(lo + CHUNK + (round ? 1 : 0), sl.w1);
                        if (it >= STAGES) mbar_wait(&sh.empty[st], (it / STAGES - 1) & 1, a.error_flag);
                        const unsigned bytes = e > b ? (e - b) * 16 : 0;
                        mbar_expect_tx(&sh.full[st], bytes);
                        if (bytes) bulk_load(sh.ring[st] + (b - lo) * 16, src + b, bytes, &sh.full[st]);
                    }
                }
            }
        }
        __syncwarp();
        if (cluster > 1) cluster_wait();
        return;
    }
    if (warp == CT / 32 + 1) {              // ---- what else a row needs ----
        const int lane = tid & 31;
        unsigned it = 0;
        for (long long n = n0; n < a.rows; n += step, ++it) {
            const int b = it & 1;
            const T* p = reinterpret_cast<const T*>(a.z) + n * a.pitch;
            const Row<T> row(p, a.v);
            const Slice sl = slice_of(row, rank, a.per);
            if (it >= 2) mbar_wait(&sh.side_empty[b], (it / 2 - 1) & 1, a.error_flag);
            if ((lane == 1 && sl.w0 == 1) || (lane == 2 && sl.tail())) {
                float x[E];
                row.part(lane == 1 ? sl.first : sl.first + sl.m - 1, x);
                (lane == 1 ? sh.edges[b].head : sh.edges[b].tail) = pack(x, T());
            }
            if constexpr (DISTILL) {
                teacher_row(sh.teach[b], p, a.v, a.te, n, a.k, c);
                if (GRAD && lane == 0) sh.weight[b] = __ldg(a.weights + n);
            } else if (lane == 0) {
                const long long t = load_id(a.ids, n, a.wide);
                const bool there = t >= 0 && t < a.v;
                sh.own[b] = {there ? to_f(__ldg(p + t)) : NEG_INF, there};
            }
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&sh.side_full[b])) : "memory");
        }
        if (cluster > 1) cluster_wait();
        return;
    }

    // ---- logits ----
    auto arrive = [&](uint64_t* bar) {      // by a warp
        __syncwarp();
        if ((tid & 31) == 0) asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
    };
    unsigned it = 0, turn = 0;
    for (long long n = n0; n < a.rows; n += step, ++turn) {
        const Row<T> row(reinterpret_cast<const T*>(a.z) + n * a.pitch, a.v);
        const Slice sl = slice_of(row, rank, a.per);
        const int b = turn & 1;
        Acc acc(c);
        acc.slot = tid < sl.m ? sl.first + tid : -1;
        for (int lo = 0; lo < sl.w1; lo += CHUNK, ++it) {
            const int st = it % STAGES;
            const uint4* chunk = reinterpret_cast<const uint4*>(sh.ring[st]);
            mbar_wait(&sh.full[st], (it / STAGES) & 1, a.error_flag);
            if (lo >= sl.w0 && lo + CHUNK <= sl.w1) {
                uint4 u[U];
#pragma unroll
                for (int q = 0; q < U; ++q) u[q] = chunk[tid + q * CT];
                arrive(&sh.empty[st]);
                take<T, ENT, TOP>(acc, u, sl.first + lo + tid, CT, c);
            } else {
                for (int s = tid; s < CHUNK; s += CT) {
                    if (lo + s < sl.w0 || lo + s >= sl.w1) continue;
                    const uint4 u[1] = {chunk[s]};
                    take<T, ENT, TOP>(acc, u, sl.first + lo + s, CT, c);
                }
                arrive(&sh.empty[st]);
            }
        }
        mbar_wait(&sh.side_full[b], (turn / 2) & 1, a.error_flag);
        // the slots over the row's ends, by the threads whose turn their places are
        if (sl.w0 == 1 && tid == 0) { float x[E]; unpack(sh.edges[b].head, x, T()); take_part<T, ENT, TOP>(acc, x, sl.first, c); }
        if (sl.tail() && tid == (sl.m - 1) % CT) { float x[E]; unpack(sh.edges[b].tail, x, T()); take_part<T, ENT, TOP>(acc, x, sl.first + sl.m - 1, c); }
        __syncwarp();

        Stat st = cta_totals<CT>(acc, sh.stat[b]);
        if constexpr (TOP) {
            const int have = top_of_cta(sh.top, acc, row, sl.first, TT, sl.first + sl.m, a.k,
                                        [&](int s, float (&x)[E]) { if (row.whole(s)) unpack(row.raw(s), x, T()); else row.part(s, x); });
            if (cluster > 1) { cluster_wait(); send_top(sh.top, have, rank); }
        } else {
            if (cluster > 1) cluster_wait();
        }
        if (cluster > 1) st = exchange<CT>(st, sh.stat[b], &sh.peers[0], cluster, rank, a.error_flag);
        Final f = {};
        if (again<T, ENT>(st.mx, c)) {
            Acc sec(c);
            for (int s = sl.first + tid; s < sl.first + sl.m; s += CT) {
                float x[E];
                if (row.whole(s)) unpack(row.raw(s), x, T()); else row.part(s, x);
                take_against<ENT>(sec, x, st.mx, c);
            }
            rows_sync<CT>();                // sh.second may still be read for the row before
            Stat st2 = cta_totals<CT>(sec, sh.second);
            if (cluster > 1) st2 = exchange<CT>(st2, sh.second, &sh.peers[1], cluster, rank, a.error_flag);
            f = finish_against(st2, st.mx);
        } else if (MODE != ROWS_LOGPROB || warp == 0) {             // without alternatives one thread writes
            f = finish(st, c);
        }

        if constexpr (!DISTILL) {
            if (rank == 0 && tid == 0) {
                const OwnLogit own = sh.own[b];
                a.out.logp[n] = !own.there ? 0.f : f.empty ? NEG_INF : (own.z - f.m) * a.scale - f.ln_s;
                a.out.lse[n] = f.m * a.scale + f.ln_s;
                a.out.entropy[n] = f.ln_s - f.mean;
            }
            if constexpr (TOP) {
                if (rank == 0) {
                    if (cluster > 1) merge_top(sh.top, cluster, a.k);
                    if (tid < a.k) {
                        const unsigned long long key = sh.top.cand[tid];
                        a.out.top[n * a.k + tid] = f.empty ? NEG_INF : (value_of((unsigned)(key >> 32)) - f.m) * a.scale - f.ln_s;
                        a.out.top_ids[n * a.k + tid] = (int)index_of(key);
                    }
                }
            }
        } else {
            const TeacherShared& teach = sh.teach[b];
            if (rank == 0 && warp == 0) {
                const float l = distill_loss(teach, f, a.k, a.scale);
                if (tid == 0) a.loss[n] = l;
            }
            if constexpr (GRAD) {
                const float w = sh.weight[b];
                const bool zero = w == 0.f || f.empty || !teach.some;
                const float up = w * a.scale, fac = up / f.s;
                // logit j at element j - base of the slice; stores along the output's own slots
                T* o = reinterpret_cast<T*>(a.g) + n * a.g_pitch;
                const int lead = (int)((reinterpret_cast<uintptr_t>(o) & 15) / sizeof(T));
                const int base = sl.first * E - row.lead, end = base + sl.w1 * E;       // [.., end): the whole slots' logits
                auto slot_at = [&](int j) { return (j + lead + E - 1) / E; };           // first output slot that begins at j or later
                for (int lo = 0; lo < sl.w1; lo += CHUNK, ++it) {
                    const int st = it % STAGES;
                    const uint4* chunk = reinterpret_cast<const uint4*>(sh.ring[st]);
                    const int from = max(lo, sl.w0), to = min(lo + CHUNK, sl.w1);
                    const int s0 = slot_at(base + from * E), s1 = to == sl.w1 ? (end + lead) / E : slot_at(base + to * E);
                    const int off = s0 * E - lead - (base + lo * E), shift = off % E * (int)sizeof(T);
                    const uint4* win = chunk + off / E;
                    uint4* dst = reinterpret_cast<uint4*>(o - lead) + s0;
                    mbar_wait(&sh.full[st], (it / STAGES) & 1, a.error_flag);
                    for (int i = tid; i < s1 - s0; i += CT) {
                        float x[E];
                        if (zero) {
#pragma unroll
                            for (int q = 0; q < E; ++q) x[q] = 0.f;
                        } else {
                            if (shift == 0) unpack(win[i], x, T()); else unpack(shifted(win[i], win[i + 1], shift), x, T());
#pragma unroll
                            for (int q = 0; q < E; ++q) x[q] = ex2((x[q] - f.m) * c) * fac;
                        }
                        dst[i] = pack(x, T());
                    }
                    arrive(&sh.empty[st]);
                }
                // logits before the first and after the last of those slots: by element
                const int j0 = max(base, 0), j1 = min(base + sl.m * E, a.v);
                const int ja = sl.w1 > sl.w0 ? slot_at(base + sl.w0 * E) * E - lead : j1, jb = sl.w1 > sl.w0 ? (end + lead) / E * E - lead : j1;
                if (tid < 4 * E) {
                    const int j = tid < 2 * E ? j0 + tid : max(jb, ja) + tid - 2 * E;
                    if (j < (tid < 2 * E ? min(ja, j1) : j1)) o[j] = from_f<T>(zero ? 0.f : ex2((to_f(__ldg(row.p + j)) - f.m) * c) * fac);
                }
                if (!zero) {
                    rows_sync<CT>();        // the dense gradient lies before the teacher's places
                    if (tid < a.k) {
                        const int id = teach.id[tid];
                        if (id >= j0 && id < j1) {
                            float q = 0.f;
                            for (int i = 0; i < a.k; ++i) q += teach.id[i] == id ? teach.q[i] : 0.f;
                            o[id] = from_f<T>(ex2((teach.z[tid] - f.m) * c) * fac - up * q);
                        }
                    }
                }
            }
        }
        arrive(&sh.side_empty[b]);
    }
}

// ---- short rows ------------------------------------------------------------------------------------
// A row of at most L * E logits lies in the registers of L lanes (logit j in lane j % L), so its maximum is known
// before the first exponential and S is 1 + the others' sum: ln S = log1p keeps its digits on confident rows.
// 65536 rows of 10: L = 4 lanes a row, 64 rows a CTA, 8 us, launch included (a CTA per row: 547).  Alternatives take a
// round of the warp each, over all registers: meant for a few.
enum { LANES_LOGPROB, LANES_GRAD, LANES_DISTILL, LANES_DISTILL_GRAD };

struct LanesArgs {
    const void* z;
    void* g;
    long long pitch, g_pitch, rows;
    int v, k;
    float scale;
    const void* ids;
    int wide;
    LogprobOut out;                                        // logprob
    const float *lse, *g_logp, *entropy, *g_entropy;       // its gradient
    Teacher te;                                            // distillation
    const float* weights;
    float* loss;
};

template <int L> __device__ __forceinline__ float lanes_max(float x) {
#pragma unroll
    for (int o = L / 2; o >= 1; o >>= 1) x = fmaxf(x, __shfl_xor_sync(~0u, x, o));
    return x;
}
template <int L> __device__ __forceinline__ float lanes_sum(float x) {
#pragma unroll
    for (int o = L / 2; o >= 1; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
    return x;
}

template <class T, int L, int E, int MODE>
__global__ void __launch_bounds__(TT) token_lanes_kernel(const LanesArgs a) {
    extern __shared__ __align__(128) unsigned char dyn[];
    const long long want = ((long long)blockIdx.x * TT + threadIdx.x) / L;
    const bool live = want < a.rows;
    const long long n = live ? want : a.rows - 1;          // lanes without a row follow the last one and store nothing
    const int lane = threadIdx.x % L;
    const T* p = reinterpret_cast<const T*>(a.z) + n * a.pitch;
    const float c = a.scale * LOG2E;
    float x[E];
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = lane + i * L < a.v ? to_f(__ldg(p + lane + i * L)) : NEG_INF;

    if (MODE == LANES_GRAD) {
        const long long t = load_id(a.ids, n, a.wide);
        const float norm = __ldg(a.lse + n), gl = t >= 0 && t < a.v ? __ldg(a.g_logp + n) : 0.f;
        const float gh = a.g_entropy ? __ldg(a.g_entropy + n) : 0.f, h = a.g_entropy ? __ldg(a.entropy + n) : 0.f;
        const bool zero = norm == NEG_INF || (gl == 0.f && gh == 0.f), far = fabsf(norm) >= FAR_LSE;
        T* g = reinterpret_cast<T*>(a.g) + n * a.g_pitch;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int j = lane + i * L;
            if (live && j < a.v) {
                float d = fmaf(x[i], a.scale, -norm);
                if (far && d > 0.f) d = 0.f;
                const float pr = ex2(d * LOG2E);
                float r = -a.scale * pr * fmaf(gh, floor_y(d) + h, gl);
                if (j == t) r += gl * a.scale;
                g[j] = from_f<T>(zero ? 0.f : r);
            }
        }
        return;
    }

    float m = x[0];
#pragma unroll
    for (int i = 1; i < E; ++i) m = fmaxf(m, x[i]);
    m = lanes_max<L>(fmaxf(m, NEG_INF));
    unsigned top = ~0u;                                    // the maximum's place, the lowest of equal ones
#pragma unroll
    for (int i = E - 1; i >= 0; --i)
        if (x[i] == m && lane + i * L < a.v) top = lane + i * L;
#pragma unroll
    for (int o = L / 2; o >= 1; o >>= 1) top = min(top, __shfl_xor_sync(~0u, top, o));
    const float ref = m == NEG_INF ? 0.f : m;
    float others = 0.f, sum_y = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const float y = (x[i] - ref) * c, e = ex2(y);
        if (lane + i * L != (int)top) {
            others += e;
            if (MODE == LANES_LOGPROB) sum_y = fmaf(e, floor_y(y), sum_y);
        }
    }
    others = lanes_sum<L>(others);
    if (m == INFINITY) others = NAN;
    const bool empty = m == NEG_INF && others == 0.f;
    const float ln_s = empty ? 0.f : log1pf(others), inv_s = 1.f / (1.f + others);

    if (MODE == LANES_LOGPROB) {
        sum_y = lanes_sum<L>(sum_y);
        if (live && lane == 0) {
            const long long t = load_id(a.ids, n, a.wide);
            const bool there = t >= 0 && t < a.v;
            a.out.logp[n] = !there ? 0.f : empty ? NEG_INF : (to_f(__ldg(p + t)) - m) * a.scale - ln_s;
            a.out.lse[n] = m * a.scale + ln_s;
            a.out.entropy[n] = empty ? 0.f : ln_s - LN2 * sum_y * inv_s;
        }
        unsigned taken = 0;
        for (int r = 0; r < a.k; ++r) {
            unsigned best = 0, at = ~0u;                   // orders of logits are above 0
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const unsigned o = lane + i * L < a.v && !(taken >> i & 1) ? order_of(x[i]) : 0;
                if (o > best) { best = o; at = lane + i * L; }
            }
            unsigned long long key = best ? key_of(best, at) : 0;
#pragma unroll
            for (int o = L / 2; o >= 1; o >>= 1) key = max(key, __shfl_xor_sync(~0u, key, o));
            const unsigned j = index_of(key);
            if (j % L == (unsigned)lane) taken |= 1u << (j / L);
            if (live && lane == r % L) {
                a.out.top[n * a.k + r] = empty ? NEG_INF : (value_of((unsigned)(key >> 32)) - m) * a.scale - ln_s;
                a.out.top_ids[n * a.k + r] = (int)j;
            }
        }
        return;
    }

    // distillation: the teacher's entries of this row in shared memory
    float* q = reinterpret_cast<float*>(dyn) + (long long)(threadIdx.x / L) * 3 * a.k;
    float* zk = q + a.k;
    int* id = reinterpret_cast<int*>(zk + a.k);
    float mu = NEG_INF;
    for (int i = lane; i < a.k; i += L) {
        const long long t = load_id(a.te.ids, n * a.k + i, a.te.wide);
        const bool there = t >= 0 && t < a.v;
        const float u = there ? a.te.value(n * a.k + i) : NEG_INF;
        q[i] = u;
        id[i] = there ? (int)t : -1;
        zk[i] = there ? to_f(__ldg(p + t)) : NEG_INF;
        mu = fmaxf(mu, u);
    }
    mu = lanes_max<L>(mu);
    if (mu == NEG_INF) mu = 0.f;
    float total = 0.f;
    for (int i = lane; i < a.k; i += L) total += ex2((q[i] - mu) * c);
    total = lanes_sum<L>(total);
    const bool some = total != 0.f;
    const float ln_total = logf(total);
    float loss = 0.f;
    for (int i = lane; i < a.k; i += L) {
        const float y = (q[i] - mu) * c, qi = some ? ex2(y) / total : 0.f;
        const float lp = empty ? NEG_INF : (zk[i] - m) * a.scale - ln_s;
        if (!(qi == 0.f)) loss += qi * ((y * LN2 - ln_total) - lp);
        q[i] = qi;
    }
    loss = lanes_sum<L>(loss);
    if (live && lane == 0) a.loss[n] = loss;
    if (MODE != LANES_DISTILL_GRAD) return;
    const float w = __ldg(a.weights + n);
    const bool zero = w == 0.f || empty || !some;
    const float up = w * a.scale, fac = up * inv_s;
    T* g = reinterpret_cast<T*>(a.g) + n * a.g_pitch;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int j = lane + i * L;
        if (live && j < a.v) g[j] = from_f<T>(zero ? 0.f : ex2((x[i] - ref) * c) * fac);
    }
    __syncwarp();                                          // q and id of all lanes; the places below are written again
    if (zero || !live) return;
    for (int i = lane; i < a.k; i += L) {
        if (id[i] < 0) continue;
        float sum = 0.f;
        for (int h = 0; h < a.k; ++h) sum += id[h] == id[i] ? q[h] : 0.f;
        g[id[i]] = from_f<T>(ex2((zk[i] - ref) * c) * fac - up * sum);
    }
}

// ---- launches --------------------------------------------------------------------------------------

template <class T> constexpr int dtype_slot() { return std::is_same<T, float>::value ? 0 : std::is_same<T, __half>::value ? 1 : 2; }

template <class A>
int launch_rows(Device* dev, void (*kernel)(A), long long blocks, int cluster, size_t smem, const A& args, int threads = TT) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = dev->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)cluster; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 1 : 0;
    EB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, args));
    count_launch();
    return EB200_OK;
}

template <class T, int MODE>
int launch_rows_of(Device* dev, const TokenShape& t, const RowsArgs& a) {
    using S = RowsShape<MODE>;
    if (!(dev->token_configured >> (MODE * 3 + dtype_slot<T>()) & 1)) {
        EB_CHECK_CUDA(cudaFuncSetAttribute(token_rows_kernel<T, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(RowsShared<MODE>)));
        dev->token_configured |= 1u << (MODE * 3 + dtype_slot<T>());
    }
    const long long ctas = t.cluster > 1 ? t.n * t.cluster : std::min(t.n, (long long)dev->prop.multiProcessorCount * S::CTAS);
    return launch_rows(dev, token_rows_kernel<T, MODE>, ctas, t.cluster, sizeof(RowsShared<MODE>), a, S::THREADS);
}

template <class T>
int launch_long(Device* dev, const Plan& plan, const void* const* in, void* const* out) {
    const TokenShape& t = plan.tok;
    const int wide = t.id_dtype == EB200_I64, esize = wide ? 8 : 4;
    auto index = [&](int i) { return (const void*)(reinterpret_cast<const char*>(in[i]) + plan.p.in[i].offset * esize); };
    RowsArgs a = {};
    a.z = reinterpret_cast<const T*>(in[0]) + t.offset;
    a.pitch = t.pitch; a.g_pitch = t.g_pitch; a.rows = t.n; a.v = t.v; a.k = t.k; a.scale = t.scale; a.wide = wide;
    a.cluster = t.cluster; a.per = t.slice; a.error_flag = dev->error_flag_dev;
    if (plan.impl == IMPL_TOKEN_LOGPROB) {
        a.ids = index(1);
        a.out = {reinterpret_cast<float*>(out[0]) + t.g_offset, reinterpret_cast<float*>(out[1]), reinterpret_cast<float*>(out[2]),
                 t.k ? reinterpret_cast<float*>(out[3]) : nullptr, t.k ? reinterpret_cast<int*>(out[4]) : nullptr};
        return t.k ? launch_rows_of<T, ROWS_TOP>(dev, t, a) : launch_rows_of<T, ROWS_LOGPROB>(dev, t, a);
    }
    a.te = {reinterpret_cast<const char*>(in[1]) + plan.p.in[1].offset * (t.teacher_dtype == EB200_F32 ? 4 : 2), index(2), t.teacher_dtype, wide};
    a.loss = reinterpret_cast<float*>(out[0]) + (t.grad ? 0 : t.g_offset);
    if (!t.grad) return launch_rows_of<T, ROWS_DISTILL>(dev, t, a);
    a.weights = reinterpret_cast<const float*>(in[3]) + plan.p.in[3].offset;
    a.g = reinterpret_cast<T*>(out[1]) + t.g_offset;
    return launch_rows_of<T, ROWS_DISTILL_GRAD>(dev, t, a);
}

template <class T, int L, int E>
int launch_lanes_of(Device* dev, const Plan& plan, const LanesArgs& a, size_t smem) {
    const long long blocks = (a.rows + TT / L - 1) / (TT / L);
    switch (plan.impl) {
        case IMPL_TOKEN_LOGPROB: return launch_rows(dev, token_lanes_kernel<T, L, E, LANES_LOGPROB>, blocks, 1, 0, a);
        case IMPL_TOKEN_LOGPROB_GRAD:
            if constexpr (L * E <= 256) return launch_rows(dev, token_lanes_kernel<T, L, E, LANES_GRAD>, blocks, 1, 0, a);
        default: break;
    }
    if (plan.tok.grad) return launch_rows(dev, token_lanes_kernel<T, L, E, LANES_DISTILL_GRAD>, blocks, 1, smem, a);
    return launch_rows(dev, token_lanes_kernel<T, L, E, LANES_DISTILL>, blocks, 1, smem, a);
}

template <class T>
int launch_lanes(Device* dev, const Plan& plan, const void* const* in, void* const* out) {
    const TokenShape& t = plan.tok;
    const int wide = t.id_dtype == EB200_I64, esize = wide ? 8 : 4;
    auto vec = [&](int i) { return reinterpret_cast<const float*>(in[i]) + plan.p.in[i].offset; };
    auto index = [&](int i) { return (const void*)(reinterpret_cast<const char*>(in[i]) + plan.p.in[i].offset * esize); };
    LanesArgs a = {};
    a.z = reinterpret_cast<const T*>(in[0]) + t.offset;
    a.pitch = t.pitch; a.g_pitch = t.g_pitch; a.rows = t.n; a.v = t.v; a.k = t.k; a.scale = t.scale; a.wide = wide;
    if (plan.impl == IMPL_DISTILL_TOPK) {
        a.te = {reinterpret_cast<const char*>(in[1]) + plan.p.in[1].offset * (t.teacher_dtype == EB200_F32 ? 4 : 2), index(2), t.teacher_dtype, wide};
        a.loss = reinterpret_cast<float*>(out[0]) + (t.grad ? 0 : t.g_offset);
        if (t.grad) { a.weights = vec(3); a.g = reinterpret_cast<T*>(out[1]) + t.g_offset; }
    } else {
        a.ids = index(1);
        if (t.grad) {
            a.lse = vec(2); a.g_logp = vec(3);
            if (t.entropy) { a.entropy = vec(4); a.g_entropy = vec(5); }
            a.g = reinterpret_cast<T*>(out[0]) + t.g_offset;
        } else {
            a.out = {reinterpret_cast<float*>(out[0]) + t.g_offset, reinterpret_cast<float*>(out[1]), reinterpret_cast<float*>(out[2]),
                     t.k ? reinterpret_cast<float*>(out[3]) : nullptr, t.k ? reinterpret_cast<int*>(out[4]) : nullptr};
        }
    }
    const size_t smem = (size_t)(TT / t.lanes) * t.k * 12;
    if (t.lanes == 4) return launch_lanes_of<T, 4, 4>(dev, plan, a, smem);
    if (t.lanes == 8) return launch_lanes_of<T, 8, 8>(dev, plan, a, smem);
    if (t.v <= 256) return launch_lanes_of<T, 32, 8>(dev, plan, a, smem);
    return launch_lanes_of<T, 32, 32>(dev, plan, a, smem);
}

template <class T>
int launch_grad(Device* dev, const Plan& plan, const void* const* in, void* const* out) {
    const TokenShape& t = plan.tok;
    const int wide = t.id_dtype == EB200_I64, esize = wide ? 8 : 4;
    auto vec = [&](int i) { return reinterpret_cast<const float*>(in[i]) + plan.p.in[i].offset; };
    constexpr int E = Pack<T>::E;
    GradArgs a = {};
    a.z = reinterpret_cast<const T*>(in[0]) + t.offset;
    a.g = reinterpret_cast<T*>(out[0]) + t.g_offset;
    a.pitch = t.pitch; a.g_pitch = t.g_pitch; a.rows = t.n; a.v = t.v; a.scale = t.scale; a.wide = wide;
    a.ids = reinterpret_cast<const char*>(in[1]) + plan.p.in[1].offset * esize;
    a.lse = vec(2); a.g_logp = vec(3);
    if (t.entropy) { a.entropy = vec(4); a.g_entropy = vec(5); }
    a.per_row = (int)(((t.v + 2LL * (E - 1)) / E + GU * TT - 1) / (GU * TT));       // at the worst alignment
    const long long blocks = t.n * a.per_row;
    EB_REQUIRE(blocks < (1LL << 31), EB200_ERR_UNSUPPORTED, "token log-probability gradient over %lld rows of %d", t.n, t.v);
    return t.entropy ? launch_rows(dev, token_logprob_grad_kernel<T, true>, blocks, 1, 0, a) : launch_rows(dev, token_logprob_grad_kernel<T, false>, blocks, 1, 0, a);
}

template <class T>
int launch_typed(Device* dev, const Plan& plan, const void* const* in, void* const* out) {
    if (plan.tok.lanes) return launch_lanes<T>(dev, plan, in, out);
    return plan.impl == IMPL_TOKEN_LOGPROB_GRAD ? launch_grad<T>(dev, plan, in, out) : launch_long<T>(dev, plan, in, out);
}

}  // namespace

// Short rows in registers: 4 lanes up to 16 logits, 8 up to 64, a warp up to 256 (the gradient) or 1024 (the rest).
// A distillation's teacher entries lie in shared memory, so many entries per row want more lanes.
// Few longer rows: the CTAs of a cluster share one, until the GPU is full or a slice has less than two slots per thread.
// Both sides of each limit, us: 65536 f32 rows of 16 / 17 logits 6.1 / 8.4, of 64 / 65 8.5 / 22.8; 16384 bf16 rows of 256 /
// 257 8.5 / 16.6 (registers of the wider shape), of 1024 / 1025 23.6 / 103, with 20 alternatives 174 / 244, distillation
// 31 / 123, with its gradient 39 / 411; token gradient of 256 / 257 8.4 / 29.  The register forms end where a lane's
// registers do; a CTA per row beyond pays its joins and barriers per row.  222 / 223 bf16 rows of 65536, clusters of two
// and none: 12.5 / 12.5.
void token_variant(TokenShape* t, int sm_count) {
    t->cluster = 1;
    t->lanes = 0;
    t->slice = 0;
    const bool logprob_grad = t->grad && !t->distill;
    if (t->v <= (logprob_grad ? 256 : 1024)) {
        t->lanes = t->v <= 16 ? 4 : t->v <= 64 ? 8 : 32;
        while (t->lanes < 32 && TT / t->lanes * t->k * 12 > 32768) t->lanes = t->lanes == 4 ? 8 : 32;
        return;
    }
    if (logprob_grad) return;
    const int e = t->dtype == EB200_F32 ? 4 : 8;
    const long long slots = ((long long)t->v + 2 * (e - 1)) / e;       // at the worst alignment
    const long long ctas = (long long)sm_count * (t->grad ? RowsShape<ROWS_DISTILL_GRAD>::CTAS : RowsShape<ROWS_LOGPROB>::CTAS);
    while (t->cluster < MAX_CLUSTER && t->n * t->cluster * 2 <= ctas && slots / (t->cluster * 2) >= 2 * TT) t->cluster *= 2;
    t->slice = (int)((slots + t->cluster - 1) / t->cluster);
}

int launch_token(Device* dev, const Plan& plan, const void* const* in, void* const* out) {
    if (plan.tok.n == 0) return EB200_OK;
    switch (plan.tok.dtype) {
        case EB200_F32: return launch_typed<float>(dev, plan, in, out);
        case EB200_F16: return launch_typed<__half>(dev, plan, in, out);
        default: return launch_typed<__nv_bfloat16>(dev, plan, in, out);
    }
}

}  // namespace eb200
