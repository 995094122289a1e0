/*
 * mzs_policy.hip — log-probabilities of given actions, entropy, log partition, top alternatives of policy rows, and
 * their gradient (include/mzsearch.h, mzs_policy_*).
 *
 * Mathematics.  Exponentials are taken in base 2 relative to the largest logit: c = inverse_temperature * log2 e,
 * d_i = c (l_i - max l), e_i = 2^d_i, s = sum e_i, t = sum e_i d_i; then log_z = max l / T + ln 2 log2 s,
 * entropy = ln 2 (log2 s - t / s), p_i = e_i / s.  A maximum that grows by D rescales s to 2^-cD s and
 * t to 2^-cD (t - cD s), so one pass over the row does.  The difference l_i - max l is taken before the product: a row
 * of the type's lowest values (a mask written as numbers) has differences of 0, where c l_i would overflow.
 */
#include "mzs_error.h"
#include "mzs_policy_plan.h"

#include <cstdint>

namespace mzs {

/* v_mul_legacy_f32: a product in which 0 times anything is 0 */
__device__ float mul_zero_wins(float a, float b) __asm("llvm.amdgcn.fmul.legacy");

namespace {

constexpr float kLn2 = 0.69314718055994530942f;
constexpr double kLog2e = 1.44269504088896340736;
constexpr float kLow = -1000.0f; /* exponents of 2 end here: 2^-1000 is 0, and 0 times a finite number stays 0 */

struct Row {
    const void* logits;
    const uint8_t* mask;
    const void* action;
    float *log_prob, *entropy, *log_z, *row_stats, *top_log_prob;
    int32_t* top_action;
    const float *grad_log_prob, *grad_entropy, *grad_log_z;
    void* grad_logits;
    int64_t rows, n, logits_stride, mask_stride, grad_stride;
    int32_t action_bytes, top;
    int32_t values; /* k_policy_row: write the forward values (else the gradient alone is wanted) */
    float scale; /* inverse_temperature              */
    float c;     /* inverse_temperature * log2 e     */
};

typedef uint32_t w4 __attribute__((ext_vector_type(4)));
typedef w4 w4_any __attribute__((aligned(2))); /* rows may start at any element */
typedef float f2 __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));

/* A logit type: kPer elements in 16 bytes.  get: element j (a constant) of 16 bytes in registers. */
template <typename T>
struct Kind;
template <>
struct Kind<float> {
    static constexpr int kPer = 4;
    static constexpr uint32_t kNone = 0xff800000u; /* -inf */
    static __device__ __forceinline__ float load(const float* p) { return *p; }
    static __device__ __forceinline__ void store(float* p, float v) { *p = v; }
    static __device__ __forceinline__ float get(const w4& v, int j) { return __uint_as_float(v[j]); }
    static __device__ __forceinline__ void keep(w4& v, const uint32_t* m) { /* a byte of m for each */
        _Pragma("unroll") for (int j = 0; j < 4; ++j) v[j] = (m[0] >> (8 * j)) & 0xffu ? v[j] : kNone;
    }
    static __device__ __forceinline__ w4 pack(const float* x) {
        return w4{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
    }
};
template <typename T>
struct Half { /* two to a word */
    static constexpr int kPer = 8;
    /* Where a byte of m is 0 the element becomes `none`: the byte's top bit is set if it is not 0, v_perm_b32 spreads two of those bits
     * over the halves of a word (selectors 8 .. 11: the signs of the four halves of its operands), v_bfi_b32 picks: two operations an
     * element, where a comparison and a selection each would be four. */
    template <uint32_t none>
    static __device__ __forceinline__ void keep_halves(w4& v, const uint32_t* m) {
        _Pragma("unroll") for (int h = 0; h < 2; ++h) {
            const uint32_t t = ((m[h] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | m[h], up = t << 8;
            const uint32_t first = __builtin_amdgcn_perm(up, t, 0x08080a0au), second = __builtin_amdgcn_perm(up, t, 0x09090b0bu);
            v[2 * h] = (v[2 * h] & first) | (none * 0x10001u & ~first);
            v[2 * h + 1] = (v[2 * h + 1] & second) | (none * 0x10001u & ~second);
        }
    }
};
template <>
struct Kind<__bf16> : Half<__bf16> {
    static constexpr uint32_t kNone = 0xff80u;
    static __device__ __forceinline__ float load(const __bf16* p) {
        return __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(p) << 16);
    }
    static __device__ __forceinline__ void store(__bf16* p, float v) { *p = (__bf16)v; }
    static __device__ __forceinline__ float get(const w4& v, int j) {
        return __uint_as_float(j & 1 ? v[j >> 1] & 0xffff0000u : v[j >> 1] << 16);
    }
    static __device__ __forceinline__ void keep(w4& v, const uint32_t* m) { keep_halves<kNone>(v, m); }
    static __device__ __forceinline__ w4 pack(const float* x) { /* v_cvt_pk_bf16_f32: nearest even, NaN kept */
        w4 v;
        _Pragma("unroll") for (int i = 0; i < 4; ++i)
            v[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{x[2 * i], x[2 * i + 1]}), b2));
        return v;
    }
};
template <>
struct Kind<_Float16> : Half<_Float16> {
    static constexpr uint32_t kNone = 0xfc00u;
    static __device__ __forceinline__ float load(const _Float16* p) { return (float)*p; }
    static __device__ __forceinline__ void store(_Float16* p, float v) { *p = (_Float16)v; }
    static __device__ __forceinline__ float get(const w4& v, int j) {
        return (float)__builtin_bit_cast(_Float16, (uint16_t)(j & 1 ? v[j >> 1] >> 16 : v[j >> 1]));
    }
    static __device__ __forceinline__ void keep(w4& v, const uint32_t* m) { keep_halves<kNone>(v, m); }
    static __device__ __forceinline__ w4 pack(const float* x) {
        w4 v;
        _Pragma("unroll") for (int i = 0; i < 4; ++i)
            v[i] = __builtin_bit_cast(uint32_t, h2{(_Float16)x[2 * i], (_Float16)x[2 * i + 1]});
        return v;
    }
};

/* x moved `by` elements down, -inf behind them (by >= kPer: nothing is left) */
template <typename T>
__device__ __forceinline__ w4 move_down(const w4& x, uint32_t by) {
    constexpr int kBits = 8 * sizeof(T);
    const uint64_t none = (kBits == 32 ? Kind<T>::kNone : Kind<T>::kNone * 0x10001u) * 0x100000001ull;
    const uint32_t bits = by < (uint32_t)Kind<T>::kPer ? by * kBits : 128u, sh = bits & 63u;
    const uint64_t lo = x[0] | ((uint64_t)x[1] << 32), hi = x[2] | ((uint64_t)x[3] << 32);
    const uint64_t a = bits == 128u ? none : bits & 64u ? hi : lo, b = bits >= 64u ? none : hi;
    const uint64_t y0 = sh ? (a >> sh) | (b << (64u - sh)) : a, y1 = sh ? (b >> sh) | (none << (64u - sh)) : b;
    return w4{(uint32_t)y0, (uint32_t)(y0 >> 32), (uint32_t)y1, (uint32_t)(y1 >> 32)};
}

/* N vectors of a row from element i on, `stride` elements apart, as they are in memory.  Every lane loads inside the row (n >= kPer): a
 * vector that the row's end cuts is loaded from n - kPer on, so that the loads go out back to back whatever the end.  l is uniform
 * over the block: scalar base, 32-bit byte offset. */
template <typename T, int N>
__device__ __forceinline__ void load_raw(const T* __restrict__ l, uint32_t i, uint32_t stride, uint32_t n, w4* x) {
    _Pragma("unroll") for (int u = 0; u < N; ++u) {
        const uint32_t at = min(i + u * stride, n - Kind<T>::kPer);
        x[u] = *reinterpret_cast<const w4_any*>(reinterpret_cast<const char*>(l) + (uint32_t)(at * sizeof(T)));
    }
}
/* what the mask forbids and what lies behind the row's end becomes -inf; cut vectors move down to where they belong */
template <typename T, int N>
__device__ __forceinline__ void dress(const uint8_t* __restrict__ mask, uint32_t i, uint32_t stride, uint32_t n, w4* x) {
    constexpr int kPer = Kind<T>::kPer;
    if (mask) {
        uint32_t m[N][kPer / 4];
        _Pragma("unroll") for (int u = 0; u < N; ++u) __builtin_memcpy(m[u], mask + min(i + u * stride, n - kPer), kPer);
        _Pragma("unroll") for (int u = 0; u < N; ++u) Kind<T>::keep(x[u], m[u]);
    }
    _Pragma("unroll") for (int u = 0; u < N; ++u)
        if (i + u * stride > n - kPer) x[u] = move_down<T>(x[u], i + u * stride - (n - kPer));
}
template <typename T, int N>
__device__ __forceinline__ void load_vecs(const T* __restrict__ l, const uint8_t* __restrict__ mask, uint32_t i, uint32_t stride, uint32_t n,
                                          w4* x) {
    load_raw<T, N>(l, i, stride, n, x);
    dress<T, N>(mask, i, stride, n, x);
}
template <typename T>
__device__ __forceinline__ w4 load_vec(const T* __restrict__ l, const uint8_t* __restrict__ mask, uint32_t i, uint32_t n) {
    w4 x;
    load_vecs<T, 1>(l, mask, i, 0, n, &x);
    return x;
}
template <typename T, bool kStream = false>
__device__ __forceinline__ void store_vec(T* __restrict__ g, uint32_t i, const w4& v) {
    w4_any* to = reinterpret_cast<w4_any*>(reinterpret_cast<char*>(g) + (uint32_t)(i * sizeof(T)));
    if constexpr (kStream) __builtin_nontemporal_store(v, to);
    else *to = v;
}

/* Wide rows of 2-byte logits at an odd element: their vectors start at the row's second logit, so that every one is 4-byte aligned (a
 * 16-byte access that is not moves 15 % less a second: 1 GiB read 202 us instead of 169), and the first logit is one
 * thread's extra. */
template <typename T>
__device__ __forceinline__ uint32_t skew_of(const T* l) { return sizeof(T) == 2 && (reinterpret_cast<uintptr_t>(l) & 2) ? 1u : 0u; }

/* one part of a row: its largest logit, and s and t relative to it */
struct Sum {
    float big, s, t;
};

__device__ __forceinline__ int64_t row_action(const Row& p, int64_t r) {
    if (!p.action) return -1;
    return p.action_bytes == 8 ? static_cast<const int64_t*>(p.action)[r] : (int64_t)static_cast<const int32_t*>(p.action)[r];
}

/* orders by value (NaN first, then +inf ... -inf; -0 = +0), then by the lower index; 0 is below every key */
__device__ __forceinline__ uint64_t rank_key(float l, uint32_t i) {
    uint32_t b = __float_as_uint(l + 0.0f);
    b = l != l ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return ((uint64_t)b << 32) | (0xffffffffu - i);
}
__device__ __forceinline__ float key_value(uint64_t key) {
    const uint32_t b = (uint32_t)(key >> 32);
    return __uint_as_float((b & 0x80000000u) ? b & 0x7fffffffu : ~b);
}

constexpr int kBlock = kPolicyBlock;
constexpr float kInf = __builtin_inff();

/* a value of another lane, word by word */
template <int kControl, typename V>
__device__ __forceinline__ V from_lane(V v) {
    uint32_t w[sizeof(V) / 4];
    __builtin_memcpy(w, &v, sizeof(V));
    _Pragma("unroll") for (uint32_t& x : w) x = (uint32_t)__builtin_amdgcn_mov_dpp((int)x, kControl, 0xf, 0xf, true);
    __builtin_memcpy(&v, w, sizeof(V));
    return v;
}
/* the values of lanes i and i ^ 16 (i ^ 32 with kRows = 2), in the same order for both */
template <int kRows, typename V>
__device__ __forceinline__ void both_lanes(V v, V& low, V& high) {
    uint32_t w[sizeof(V) / 4], l[sizeof(V) / 4], h[sizeof(V) / 4];
    __builtin_memcpy(w, &v, sizeof(V));
    _Pragma("unroll") for (size_t i = 0; i < sizeof(V) / 4; ++i) {
        const auto two = kRows == 1 ? __builtin_amdgcn_permlane16_swap(w[i], w[i], false, false)
                                    : __builtin_amdgcn_permlane32_swap(w[i], w[i], false, false);
        l[i] = two[0], h[i] = two[1];
    }
    __builtin_memcpy(&low, l, sizeof(V));
    __builtin_memcpy(&high, h, sizeof(V));
}
/* Butterfly over G consecutive lanes: every lane gets the same bits (at each step both partners combine the same two values). */
template <int G, typename V, typename F>
__device__ __forceinline__ V lanes_reduce(V v, F op) {
    if (G > 1) v = op(v, from_lane<0xB1>(v));  /* lane ^ 1 */
    if (G > 2) v = op(v, from_lane<0x4E>(v));  /* lane ^ 2 */
    if (G > 4) v = op(v, from_lane<0x141>(v)); /* the other four of eight */
    if (G > 8) v = op(v, from_lane<0x140>(v)); /* the other eight of 16 */
    V low, high;
    if (G > 16) both_lanes<1>(v, low, high), v = op(low, high);
    if (G > 32) both_lanes<2>(v, low, high), v = op(low, high);
    return v;
}
template <int G>
__device__ __forceinline__ float lanes_max(float v) {
    return lanes_reduce<G>(v, [](float a, float b) { return fmaxf(a, b); });
}
template <int G>
__device__ __forceinline__ float lanes_sum(float v) {
    return lanes_reduce<G>(v, [](float a, float b) { return a + b; });
}

/* rank_key of a row of at most kRankMost logits in a register that one instruction compares: what the type's ranks differ in, then the inverted index.  next:
 * the largest key below `last` in the team.  Fp32 (32 + 11 bits): as the mantissa of doubles, whose maximum is one instruction; 2-byte types
 * (16 or 19 + 11 bits): key - last wraps for the keys below `last` and is largest for the nearest of them, so a maximum of differences finds it. */
constexpr uint32_t kRankMost = MZS_POLICY_NARROW;
template <typename T>
struct Rank {
    typedef uint32_t Key;
    static constexpr uint32_t kDrop = sizeof(T) == 2 && Kind<T>::kNone == 0xff80u ? 16 : 13; /* low bits of the rank that say nothing */
    static __device__ __forceinline__ Key first() { return 0x80000000u; }
    static __device__ __forceinline__ Key make(float x, uint32_t i) {
        return x == -kInf ? 0u : ((uint32_t)(rank_key(x, 0) >> 32) >> kDrop) * kRankMost + (kRankMost - 1 - i);
    }
    static __device__ __forceinline__ uint64_t whole(Key k) {
        const uint32_t rank = k / kRankMost << kDrop;
        return k == 0 ? 0 : (uint64_t)(rank | (rank & 0x80000000u ? 0u : (1u << kDrop) - 1u)) << 32 | (0xffffffffu - (kRankMost - 1 - k % kRankMost));
    }
    template <int G, int E>
    static __device__ __forceinline__ Key next(const Key* key, Key last) {
        Key best = 0u - last; /* nothing: key 0 */
        _Pragma("unroll") for (int j = 0; j < E; ++j) best = max(best, key[j] - last);
        best = lanes_reduce<G>(best, larger);
        return last == 0 ? 0 : best + last;
    }
    static __device__ __forceinline__ Key larger(Key a, Key b) { return max(a, b); }
    static __device__ __forceinline__ Key smaller(Key a, Key b) { return min(a, b); }
};
template <>
struct Rank<float> {
    typedef double Key;
    static __device__ __forceinline__ Key first() { return __longlong_as_double(0x7ff0000000000000ll); }
    static __device__ __forceinline__ Key make(float x, uint32_t i) {
        const uint64_t k = (uint64_t)(uint32_t)(rank_key(x, 0) >> 32) * kRankMost + (kRankMost - 1 - i);
        return x == -kInf ? 0.0 : __longlong_as_double((long long)(k | 0x4000000000000000ull));
    }
    static __device__ __forceinline__ uint64_t whole(Key key) {
        const uint64_t k = (uint64_t)__double_as_longlong(key) & 0x000fffffffffffffull;
        return key == 0.0 ? 0 : k / kRankMost << 32 | (0xffffffffu - (kRankMost - 1 - (uint32_t)(k % kRankMost)));
    }
    static __device__ __forceinline__ Key larger(Key a, Key b) { /* neither is ever NaN: fmax would make sure of it first */
        Key v;
        asm("v_max_f64 %0, %1, %2" : "=v"(v) : "v"(a), "v"(b));
        return v;
    }
    static __device__ __forceinline__ Key smaller(Key a, Key b) {
        Key v;
        asm("v_min_f64 %0, %1, %2" : "=v"(v) : "v"(a), "v"(b));
        return v;
    }
    template <int G, int E>
    static __device__ __forceinline__ Key next(const Key* key, Key last) {
        Key best = 0.0;
        _Pragma("unroll") for (int j = 0; j < E; ++j) best = larger(best, key[j] < last ? key[j] : 0.0);
        return lanes_reduce<G>(best, larger);
    }
};

/* From |c big| = kHuge on a row takes its exponents as c (l_i - big).  Below, they are c l_i - m with one rounding, m = c big rounded, and
 * delta = c big - m, at most half a step of m, is put right by 2^-delta: that has to stay near 1, and is, up to 2^24 (delta <= 1/2), where it
 * would be 0 or infinity from 2^34 on.  Rows up there are those of large numbers written as a mask (-1e9 everywhere) or of temperatures
 * below about 1e-6. */
constexpr float kHuge = 0x1p24f;
__device__ __forceinline__ bool is_huge(const Row& p, float big) { return !(fabsf(p.c * big) < kHuge); }

/* exponent of 2 for a logit x beside the row's largest one; finite, so that 0 * it is 0 */
__device__ __forceinline__ float exponent_of(const Row& p, float x, float big) { return fmaxf(p.c * (x - big), kLow); }
/* 2^d; a NaN logit (which fmaxf turned into kLow) stays one */
__device__ __forceinline__ float power_of(float d, float x) { return x != x ? x : __builtin_amdgcn_exp2f(d); }

struct Values {
    float log_z, entropy, log_total, log2_s;
    bool empty;
};
__device__ __forceinline__ Values row_values(const Row& p, const Sum& v) {
    Values o;
    o.empty = v.s == 0.0f;
    o.log2_s = log2f(v.s);
    o.log_total = kLn2 * o.log2_s;
    o.log_z = o.empty ? -kInf : p.scale * v.big + o.log_total;
    o.entropy = o.empty ? 0.0f : kLn2 * (o.log2_s - v.t / v.s);
    return o;
}
__device__ __forceinline__ void write_row(const Row& p, int64_t r, const Sum& v, const Values& o, float l_action, int64_t a) {
    p.log_z[r] = o.log_z;
    p.entropy[r] = o.entropy;
    p.row_stats[2 * r] = v.big;
    p.row_stats[2 * r + 1] = v.s;
    float lp = 0.0f;
    if (a >= p.n) lp = __builtin_nanf("");
    else if (a >= 0) lp = o.empty ? -kInf : p.scale * (l_action - v.big) - o.log_total;
    p.log_prob[r] = lp;
}
template <typename T>
__device__ __forceinline__ float action_logit(const Row& p, const T* l, const uint8_t* mask, int64_t a) {
    return a < 0 || a >= p.n ? 0.0f : mask && !mask[a] ? -kInf : Kind<T>::load(l + a);
}
__device__ __forceinline__ int32_t top_action(uint64_t key) { return key ? (int32_t)(0xffffffffu - (uint32_t)key) : -1; }
__device__ __forceinline__ float top_log_prob(const Row& p, uint64_t key, const Sum& v, const Values& o) {
    return key ? p.scale * (key_value(key) - v.big) - o.log_total : -kInf;
}
__device__ __forceinline__ void write_top(const Row& p, int64_t r, int k, uint64_t key, const Sum& v, const Values& o) {
    p.top_action[r * p.top + k] = top_action(key);
    p.top_log_prob[r * p.top + k] = top_log_prob(p, key, v, o);
}

/* What the gradient of a row needs: grad_i = 2^(c l_i - m) (base + slope (c l_i - m)), + at_action where i is the action. */
struct Slope {
    float big, m, base, slope, at_action;
    bool empty;
};
__device__ __forceinline__ Slope row_slope(const Row& p, int64_t r, int64_t a, const Sum& v, float entropy, float log2_s) {
    const float ga = a < 0 || !p.grad_log_prob ? 0.0f : a >= p.n ? __builtin_nanf("") : p.grad_log_prob[r];
    const float gh = p.grad_entropy ? p.grad_entropy[r] : 0.0f, gz = p.grad_log_z ? p.grad_log_z[r] : 0.0f;
    Slope q;
    q.big = v.big;
    q.m = p.c * v.big;
    const float delta = is_huge(p, v.big) ? 0.0f : fmaf(p.c, v.big, -q.m);
    const float f = p.scale / v.s * __builtin_amdgcn_exp2f(-delta); /* log p_i = ln 2 (c l_i - m - delta - log2 s) */
    q.base = f * (gz - ga - gh * (entropy - kLn2 * (log2_s + delta)));
    q.slope = f * (-gh * kLn2);
    q.at_action = p.scale * ga;
    q.empty = v.s == 0.0f;
    return q;
}
/* any logit, whatever the row (a huge one has m = 0 in effect: its exponents are differences of logits) */
__device__ __forceinline__ float slope_at(const Row& p, const Slope& q, float x) {
    const float d = is_huge(p, q.big) ? exponent_of(p, x, q.big) : fmaxf(fmaf(p.c, x, -q.m), kLow);
    return power_of(d, x) * (q.base + q.slope * d);
}
/* whether the short form of the gradient does for the row: c l_i - m as one fma, no element needs a look of its own */
__device__ __forceinline__ bool is_plain(const Row& p, const Slope& q) {
    return !q.empty && !is_huge(p, q.big) && fabsf(q.base) < kInf && fabsf(q.slope) < kInf;
}

/* Alternatives of a row whose team holds all its keys: the next one below the last, `top` times; the team's lanes write one each.  Where
 * many are asked of many lanes, each of which then has one of them or none as a rule, they are looked for among the lanes' four largest, and
 * anew among all keys if a lane's four were all taken (40000 x 1000 fp32 with 32 of them 217 -> 161 us, with 12 103 -> 76; 80000 x 1000 bf16
 * with 32 233 -> 191, with 9 109 -> 101; fewer are not worth the sorting). */
template <typename T, int kTeam, int E>
__device__ __forceinline__ void write_best(const Row& p, int64_t r, int lane, const typename Rank<T>::Key* key, const Sum& v, const Values& o) {
    typename Rank<T>::Key last = Rank<T>::first(), mine = last;
    int k = 0; /* chosen already */
    if constexpr (kTeam == 1) { /* four to a store: 2M rows of 8 with all 8 of them 66 us, one at a time 98 */
        for (; k + 4 <= p.top; k += 4) {
            w4_any at, lp;
            _Pragma("unroll") for (int i = 0; i < 4; ++i) {
                last = Rank<T>::template next<1, E>(key, last);
                const uint64_t whole = Rank<T>::whole(last);
                at[i] = (uint32_t)top_action(whole), lp[i] = __float_as_uint(top_log_prob(p, whole, v, o));
            }
            *reinterpret_cast<w4_any*>(p.top_action + r * p.top + k) = at;
            *reinterpret_cast<w4_any*>(p.top_log_prob + r * p.top + k) = lp;
        }
    }
    const auto choose = [&](const auto& keys, auto count) {
        for (int i = k; i < p.top; ++i) {
            last = Rank<T>::template next<kTeam, decltype(count)::value>(keys, last);
            const int turn = i % kTeam;
            if (turn == lane) mine = last;
            if ((turn == kTeam - 1 || i + 1 == p.top) && lane <= turn) write_top(p, r, i - turn + lane, Rank<T>::whole(mine), v, o);
        }
    };
    if constexpr (kTeam >= 32 && E >= 12) {
        if (p.top > 8 && 2 * p.top <= kTeam) {
            typename Rank<T>::Key own[4] = {}; /* the lane's four largest */
            _Pragma("unroll") for (int j = 0; j < E; ++j) {
                typename Rank<T>::Key x = key[j];
                _Pragma("unroll") for (int h = 0; h < 4; ++h) {
                    const typename Rank<T>::Key large = Rank<T>::larger(own[h], x);
                    x = Rank<T>::smaller(own[h], x), own[h] = large;
                }
            }
            choose(own, std::integral_constant<int, 4>());
            if (lanes_reduce<kTeam>(own[3] != 0 && own[3] >= last ? 1u : 0u, [](uint32_t a, uint32_t b) { return a | b; }) == 0) return;
            last = Rank<T>::first();
        }
    }
    choose(key, std::integral_constant<int, E>());
}

/* ------------------------------------------------------------------ narrow rows
 * Up to 8 logits: a lane a row, in registers; one read, one write, nothing shared.  Bound by memory: 2M x 4 fp32 with the best action
 * 20 us, 4.5 TB/s of what it reads and writes; 4096 rows 3.3 us, of which an empty launch is 2.5. */
template <typename T, int E, bool kForward, bool kGrad, bool kTop>
__global__ void __launch_bounds__(kBlock) k_policy_lanes(const Row p) {
    const int n = (int)p.n;
    for (int64_t r = (int64_t)blockIdx.x * kBlock + threadIdx.x; r < p.rows; r += (int64_t)gridDim.x * kBlock) {
        const T* l = static_cast<const T*>(p.logits) + r * p.logits_stride;
        const uint8_t* mask = p.mask ? p.mask + r * p.mask_stride : nullptr;
        const int64_t a = row_action(p, r);
        float x[E];
        _Pragma("unroll") for (int i = 0; i < E; ++i) x[i] = i < n ? Kind<T>::load(l + i) : -kInf;
        if (mask) {
            _Pragma("unroll") for (int i = 0; i < E; ++i) if (i < n && !mask[i]) x[i] = -kInf;
        }
        const float la = kForward ? action_logit<T>(p, l, mask, a) : 0.0f;
        Sum v{-kInf, 0.0f, 0.0f};
        _Pragma("unroll") for (int i = 0; i < E; ++i) v.big = fmaxf(v.big, x[i]);
        if (v.big > -kInf) {
            _Pragma("unroll") for (int i = 0; i < E; ++i) {
                const float d = exponent_of(p, x[i], v.big), e = power_of(d, x[i]);
                v.s += e, v.t = fmaf(e, d, v.t);
            }
        } else { /* nothing allowed, or nothing but NaN */
            _Pragma("unroll") for (int i = 0; i < E; ++i) if (x[i] != x[i]) v.s = x[i];
        }
        if (v.big == kInf) v.s = __builtin_nanf("");
        const Values o = row_values(p, v);
        if (kForward) write_row(p, r, v, o, la, a);
        if constexpr (kTop) {
            typename Rank<T>::Key key[E];
            _Pragma("unroll") for (int i = 0; i < E; ++i) key[i] = Rank<T>::make(x[i], (uint32_t)i);
            write_best<T, 1, E>(p, r, 0, key, v, o);
        }
        if (kGrad) {
            const Slope q = row_slope(p, r, a, v, o.entropy, o.log2_s);
            T* out = static_cast<T*>(p.grad_logits) + r * p.grad_stride;
            _Pragma("unroll") for (int i = 0; i < E; ++i) {
                float y = 0.0f;
                if (!q.empty && x[i] != -kInf) {
                    y = slope_at(p, q, x[i]);
                    if (i == a) y += q.at_action;
                }
                if (i < n) Kind<T>::store(out + i, y);
            }
        }
    }
}

/* ------------------------------------------------------------------ wide rows
 * A block walks a chunk of a row: thread t takes the 16-byte vectors t, t + kBlock, ... of it. */

/* A team of threads works on a row: some lanes of a wave, a wave, or a whole block.  Merges every thread's part; all threads return the
 * same bits.  lds: three floats a wave (a block's team) */
template <int kTeam>
__device__ __forceinline__ Sum team_merge(const Row& p, Sum v, float* lds) {
    constexpr int kWaves = kTeam / 64, kLanes = kTeam < 64 ? kTeam : 64;
    const int wave = threadIdx.x >> 6;
    const bool first = (threadIdx.x & 63) == 0;
    float big = lanes_max<kLanes>(v.big);
    if constexpr (kWaves > 1) {
        if (first) lds[wave] = big;
        __syncthreads();
        _Pragma("unroll") for (int w = 0; w < kWaves; ++w) big = fmaxf(big, lds[w]);
    }
    const float d = v.big == big ? 0.0f : fmaxf(p.c * (v.big - big), kLow), f = __builtin_amdgcn_exp2f(d);
    Sum o{big, lanes_sum<kLanes>(f * v.s), lanes_sum<kLanes>(f * (v.t + d * v.s))};
    if constexpr (kWaves > 1) {
        if (first) lds[kWaves + wave] = o.s, lds[2 * kWaves + wave] = o.t;
        __syncthreads();
        o.s = o.t = 0.0f;
        _Pragma("unroll") for (int w = 0; w < kWaves; ++w) o.s += lds[kWaves + w], o.t += lds[2 * kWaves + w];
    }
    if (big == kInf) o.s = __builtin_nanf("");
    return o;
}

constexpr int kAhead = kPolicyAhead; /* vectors a thread has in flight */

/* The compiler may not look behind this: a row held packed is unpacked anew in each pass over it, where it would otherwise keep every
 * unpacked value (twice the registers, which spill). */
__device__ __forceinline__ void unpack_here(w4& v) { asm volatile("" : "+v"(v)); }

template <typename T, int N>
__device__ __forceinline__ float max_vecs(const w4* v, float big) {
    _Pragma("unroll") for (int u = 0; u < N; ++u)
        _Pragma("unroll") for (int j = 0; j < Kind<T>::kPer; ++j) big = fmaxf(big, Kind<T>::get(v[u], j));
    return big;
}
/* A thread's running sum over the vectors of a wide row, relative to m = c * big held within +-kReach: the exponent is one fma, c l_i - m
 * with a single rounding, and what m lost to its own rounding is put right once at the end.  Where m was held above, the row is huge and
 * summed again by sum_slowly; where it was held below, either all of the row is as low and huge too, or the row's largest logit is at least
 * 2^24 above in exponents and what this thread has counts for nothing (kReach is twice kHuge for that: a part that lies a little below
 * a row that is just not huge still has its own m). */
constexpr float kReach = 2.0f * kHuge;
struct Running {
    float big, m, s, t;
};
__device__ __forceinline__ Running running_start() { return Running{-kInf, -kReach, 0.0f, 0.0f}; }

/* takes N vectors: their maximum first, one rescaling, then the exponentials */
template <typename T, int N>
__device__ __forceinline__ void take_vecs(const Row& p, const w4* v, Running& sum) {
    const float big = max_vecs<T, N>(v, sum.big), m = __builtin_amdgcn_fmed3f(p.c * big, -kReach, kReach);
    const float shift = fmaxf(sum.m - m, kLow), f = __builtin_amdgcn_exp2f(shift);
    float s = f * sum.s, t = f * (sum.t + shift * sum.s);
    _Pragma("unroll") for (int u = 0; u < N; ++u)
        _Pragma("unroll") for (int j = 0; j < Kind<T>::kPer; ++j) {
            const float d = fmaf(p.c, Kind<T>::get(v[u], j), -m), e = __builtin_amdgcn_exp2f(d);
            s += e, t = fmaf(e, fmaxf(d, kLow), t);
        }
    sum = Running{big, m, s, t};
}
/* takes one logit */
__device__ __forceinline__ void take_one(const Row& p, float x, Running& sum) {
    const float big = fmaxf(sum.big, x), m = __builtin_amdgcn_fmed3f(p.c * big, -kReach, kReach);
    const float shift = fmaxf(sum.m - m, kLow), f = __builtin_amdgcn_exp2f(shift);
    const float d = fmaf(p.c, x, -m), e = __builtin_amdgcn_exp2f(d);
    sum = Running{big, m, f * sum.s + e, fmaf(e, fmaxf(d, kLow), f * (sum.t + shift * sum.s))};
}
/* the same relative to big itself, where m was not held */
__device__ __forceinline__ Sum running_end(const Row& p, const Running& v) {
    const float delta = fabsf(v.m) < kReach ? fmaf(p.c, v.big, -v.m) : 0.0f, f = __builtin_amdgcn_exp2f(-delta);
    return Sum{v.big, f * v.s, f * (v.t - delta * v.s)};
}
/* this thread's vectors i, i + stride, ... and its extra logit (-inf: none) of a row whose largest logit `big` is huge */
template <typename T>
__device__ Sum sum_slowly(const Row& p, const T* l, const uint8_t* mask, uint32_t i, uint32_t stride, uint32_t end, uint32_t n, float big,
                          float extra) {
    Sum v{big, 0.0f, 0.0f};
    {
        const float d = exponent_of(p, extra, big), e = power_of(d, extra);
        v.s += e, v.t = fmaf(e, d, v.t);
    }
    for (; i < end && i < n; i += stride) {
        const w4 x = load_vec<T>(l, mask, i, n);
        _Pragma("unroll") for (int j = 0; j < Kind<T>::kPer; ++j) {
            const float y = Kind<T>::get(x, j), d = exponent_of(p, y, big), e = power_of(d, y);
            v.s += e, v.t = fmaf(e, d, v.t);
        }
    }
    return v;
}

constexpr int kStrips = 512; /* strips that can hold alternatives              */
constexpr int kKeys = 1024;  /* logits that can be alternatives                */
constexpr int kGroups = kBlock / 4; /* four threads' strips: enough groups for MZS_POLICY_MAX_TOP of them */
static_assert(kGroups == 64 && MZS_POLICY_MAX_TOP <= kGroups, "tau is one of the groups' maxima, a lane's each");
struct TopScratch {
    uint64_t keys[kKeys];
    uint32_t strips[kStrips];
    alignas(16) uint32_t groups[kGroups];
    uint32_t n_strips, n_keys, tau;
    uint64_t best[kBlock / 64];
};

/* order of logits as unsigned numbers, 0 for what is not allowed */
__device__ __forceinline__ uint32_t rank_value(float x) { return x == -kInf ? 0u : (uint32_t)(rank_key(x, 0) >> 32); }

constexpr int kStripLanes = kPolicyStripLanes, kStripsPerBlock = kPolicyStrips;
constexpr int kHold = 16; /* strips of a row that a thread holds in registers */
/* strip in held[h] of this thread; >= n_strips: none.  Few strips are spread over the block, so that every group has one. */
__device__ __forceinline__ int held_strip(int h, int n_strips) {
    const int spread = n_strips <= kBlock / 4 ? 4 : n_strips <= kBlock / 2 ? 2 : 1;
    const int at = threadIdx.x + h * kBlock;
    return at % spread ? n_strips : at / spread;
}

/* Alternatives from strips.  A strip is the vectors that kLanes neighbouring threads took of one chunk; its largest logit is known.  Each
 * four of the block's threads take the largest over their share of the strips; tau, the top-th largest of those 64, is reached by at least
 * `top` logits, so
 *   1. strips whose maximum reaches tau are read again and their logits that reach it collected — hardly more than `top` of them, as
 *      the best ones seldom share a group (top 20: 24 on the average, top 32: 44);
 *   2. a collected logit's rank is the number of collected ones before it.
 * Both need little more than the strips' maxima, whatever the logits — unless many are alike: where they do not
 * fit the lists, only those above tau are collected, and the ones equal to tau are taken from the row's start on.  A row where
 * even that is too much (or with NaN) is searched `top` times.  Every choice is by value and index: the lists' order does not matter.
 * A row that one block has whole knows its threads' own maxima (kLanes 1: a 256th of the row for each alternative is read again); strips
 * that travel through memory to the join are four threads' each (a 64th of what the block took). */
template <typename T, int kLanes, int kHeld, typename Maximum>
__device__ void select_top(const Row& p, int64_t r, const T* l, const uint8_t* mask, const Sum& v, const Values& o, const float* held, Maximum maximum,
                           int n_strips, int chunk_vecs, uint32_t chunk_len, TopScratch& sh) {
    constexpr int kPer = Kind<T>::kPer;
    constexpr uint32_t kPerBlock = kBlock / kLanes;
    const int tid = threadIdx.x;
    const uint32_t want = (uint32_t)p.top, n = (uint32_t)p.n;
    const bool plain = v.s == v.s;
    uint32_t mine = 0;
    _Pragma("unroll") for (int h = 0; h < kHeld; ++h) mine = max(mine, rank_value(held[h]));
    for (int i = tid + kHeld * kBlock; i < n_strips; i += kBlock) mine = max(mine, rank_value(maximum(i)));
    const uint32_t group = lanes_reduce<4>(mine, [](uint32_t a, uint32_t b) { return max(a, b); });
    if (tid % 4 == 0) sh.groups[tid / 4] = group;
    if (tid == 0) sh.n_strips = 0, sh.n_keys = 0;
    __syncthreads();
    if (tid < kGroups) { /* a wave */
        const uint32_t g = sh.groups[tid];
        uint32_t ahead = 0; /* groups with a larger one */
        _Pragma("unroll") for (int i = 0; i < kGroups; ++i) ahead += (uint32_t)__builtin_amdgcn_readlane((int)g, i) > g;
        const uint32_t least = lanes_reduce<kGroups>(ahead < want ? g : 0xffffffffu, [](uint32_t a, uint32_t b) { return min(a, b); });
        if (tid == 0) sh.tau = least; /* the smallest of those that fewer than `top` are ahead of */
    }
    bool done = false;
    for (int stage = 0; stage < 2 && plain && !done; ++stage) {
        __syncthreads();
        const uint32_t tau = sh.tau, least = stage ? tau + 1u : max(tau, 1u);
        if (stage) {
            if (tid == 0) sh.n_strips = 0, sh.n_keys = 0;
            __syncthreads();
        }
        const auto look = [&](float largest, int i) {
            if (rank_value(largest) >= least) {
                const uint32_t at = atomicAdd(&sh.n_strips, 1u);
                if (at < kStrips) sh.strips[at] = i;
            }
        };
        if (mine >= least) {
            _Pragma("unroll") for (int h = 0; h < kHeld; ++h) look(held[h], kLanes == 1 ? tid : held_strip(h, n_strips));
            for (int i = tid + kHeld * kBlock; i < n_strips; i += kBlock) look(maximum(i), i);
        }
        __syncthreads();
        const uint32_t found = sh.n_strips, each = (uint32_t)chunk_vecs * kLanes;
        if (found <= kStrips) {
            for (uint32_t w = tid; w < found * each; w += kBlock) {
                const uint32_t strip = sh.strips[w / each], lane = w % kLanes, j = w % each / kLanes;
                const uint32_t i = skew_of(l) + strip / kPerBlock * chunk_len + (j * kBlock + strip % kPerBlock * kLanes + lane) * kPer;
                if (i >= n) continue;
                const w4 x = load_vec<T>(l, mask, i, n);
                _Pragma("unroll") for (int q = 0; q < kPer; ++q) {
                    const uint32_t k = rank_value(Kind<T>::get(x, q));
                    if (k >= least) {
                        const uint32_t at = atomicAdd(&sh.n_keys, 1u);
                        if (at < kKeys) sh.keys[at] = ((uint64_t)k << 32) | (0xffffffffu - (i + q));
                    }
                }
            }
            if (tid == 0 && skew_of(l)) { /* the row's extra logit */
                const uint32_t k = rank_value(action_logit<T>(p, l, mask, 0));
                if (k >= least) {
                    const uint32_t at = atomicAdd(&sh.n_keys, 1u);
                    if (at < kKeys) sh.keys[at] = ((uint64_t)k << 32) | 0xffffffffu;
                }
            }
        }
        __syncthreads();
        const uint32_t n_keys = sh.n_keys;
        done = found <= kStrips && n_keys <= kKeys;
        if (done) {
            for (uint32_t i = tid; i < n_keys; i += kBlock) {
                const uint64_t key = sh.keys[i];
                uint32_t rank = 0;
                for (uint32_t k = 0; k < n_keys; ++k) rank += sh.keys[k] > key;
                if (rank < want) write_top(p, r, rank, key, v, o);
            }
            uint32_t at = min(n_keys, want);
            if (stage && tau) { /* equal ones in the row's order */
                for (uint32_t i0 = 0; i0 < n && at < want; i0 += kBlock * kPer) {
                    const uint32_t i = i0 + tid * kPer;
                    uint32_t hit = 0;
                    if (i < n) {
                        const w4 x = load_vec<T>(l, mask, i, n);
                        _Pragma("unroll") for (int q = 0; q < kPer; ++q) hit |= (uint32_t)(rank_value(Kind<T>::get(x, q)) == tau) << q;
                    }
                    const uint32_t count = __popc(hit);
                    uint32_t up_to = count;
                    for (int off = 1; off < 64; off <<= 1) {
                        const uint32_t other = __shfl_up(up_to, off, 64);
                        if ((tid & 63) >= off) up_to += other;
                    }
                    if ((tid & 63) == 63) sh.groups[tid >> 6] = up_to;
                    __syncthreads();
                    uint32_t slot = at + up_to - count, all = 0;
                    for (int w = 0; w < kBlock / 64; ++w) {
                        if (w < (tid >> 6)) slot += sh.groups[w];
                        all += sh.groups[w];
                    }
                    for (int q = 0; q < kPer; ++q)
                        if ((hit >> q) & 1u) {
                            if (slot < want) write_top(p, r, slot, ((uint64_t)tau << 32) | (0xffffffffu - (i + q)), v, o);
                            ++slot;
                        }
                    at = min(at + all, want);
                    __syncthreads();
                }
            }
            for (uint32_t k = at + tid; k < want; k += kBlock) write_top(p, r, k, 0, v, o);
        }
    }
    if (done) return;
    uint64_t last = ~0ull;
    for (uint32_t k = 0; k < want; ++k) {
        uint64_t best = 0;
        for (uint32_t i = tid * kPer; i < n; i += kBlock * kPer) {
            const w4 x = load_vec<T>(l, mask, i, n);
            _Pragma("unroll") for (int q = 0; q < kPer; ++q) {
                const uint32_t c = rank_value(Kind<T>::get(x, q));
                const uint64_t key = c ? ((uint64_t)c << 32) | (0xffffffffu - (i + q)) : 0;
                if (key < last && key > best) best = key;
            }
        }
        for (int off = 1; off < 64; off <<= 1) {
            const uint64_t other = __shfl_xor((unsigned long long)best, off, 64);
            best = other > best ? other : best;
        }
        __syncthreads();
        if ((tid & 63) == 0) sh.best[tid >> 6] = best;
        __syncthreads();
        for (int w = 0; w < kBlock / 64; ++w) best = max(best, sh.best[w]);
        last = best;
        if (tid == 0) write_top(p, r, k, last, v, o);
    }
}

/* Forward pass of a chunk: one read, running maximum and sums, four vectors a thread on their way while four are summed.  kSplit: the
 * chunk's part goes to parts[row][chunk] and its strips' maxima to strips[row][chunk][strip]; else the chunk is the row.  Bound by the read
 * and the arithmetic alike: an element's eight operations and its exponential, which takes four places, are 19.5 us of the card's lanes for 64M
 * elements, the read of 640 x 100000 bf16 19.7, and with 2.5 waves a SIMD the two overlap in part: 30 to 34 us from memory, 4.2 TB/s, 37 to 39
 * with the five best alternatives, whose search every block ends with at once; two vectors in flight 30, six 33, at least six waves a SIMD
 * (fewer registers) 33. */
template <typename T, bool kSplit>
__global__ void __launch_bounds__(kBlock) k_policy_chunk(const Row p, int chunks, int chunk_vecs, float* __restrict__ parts,
                                                         float* __restrict__ strips) {
    constexpr int kPer = Kind<T>::kPer;
    __shared__ float lds[3 * (kBlock / 64)];
    const int64_t r = blockIdx.x / chunks;
    const int chunk = blockIdx.x % chunks;
    const T* l = static_cast<const T*>(p.logits) + r * p.logits_stride;
    const uint8_t* mask = p.mask ? p.mask + r * p.mask_stride : nullptr;
    const uint32_t n = (uint32_t)p.n;
    const uint32_t skew = skew_of(l), chunk_len = (uint32_t)chunk_vecs * kBlock * kPer;
    const uint32_t from = skew + chunk * chunk_len + threadIdx.x * kPer;
    const float extra = skew && from == skew ? action_logit<T>(p, l, mask, 0) : -kInf;
    const int64_t a = kSplit ? -1 : row_action(p, r); /* asked for early: nothing waits for it behind the sums */
    const float la = kSplit ? 0.0f : action_logit<T>(p, l, mask, a);
    Running sum = running_start();
    constexpr uint32_t kStride = kBlock * kPer;
    const int groups = chunk_vecs / kAhead; /* the next group is on its way while one is summed */
    w4 x[kAhead], y[kAhead];
    const auto load = [&](int g, w4* v) { if (g < groups) load_raw<T, kAhead>(l, from + (uint32_t)g * kAhead * kStride, kStride, n, v); };
    const auto take = [&](int g, w4* v) {
        dress<T, kAhead>(mask, from + (uint32_t)g * kAhead * kStride, kStride, n, v);
        take_vecs<T, kAhead>(p, v, sum);
    };
    const auto rest = [&](auto count) { /* what the groups leave, together */
        constexpr int N = decltype(count)::value;
        const uint32_t i = from + (uint32_t)groups * kAhead * kStride;
        w4 z[N];
        load_vecs<T, N>(l, mask, i, kStride, n, z);
        take_vecs<T, N>(p, z, sum);
    };
    load(0, x);
    static_assert(kAhead == 4, "a case for each rest");
    switch (chunk_vecs % kAhead) {
        case 1: rest(std::integral_constant<int, 1>()); break;
        case 2: rest(std::integral_constant<int, 2>()); break;
        case 3: rest(std::integral_constant<int, 3>()); break;
    }
    for (int g = 0; g < groups; g += 2) {
        load(g + 1, y);
        take(g, x);
        load(g + 2, x);
        if (g + 1 < groups) take(g + 1, y);
    }
    if (skew && from == skew) take_one(p, extra, sum);
    Sum v = team_merge<kBlock>(p, running_end(p, sum), lds);
    if (is_huge(p, v.big) && fabsf(v.big) < kInf) {
        __syncthreads();
        v = team_merge<kBlock>(p, sum_slowly<T>(p, l, mask, from, kBlock * kPer, skew + (chunk + 1) * chunk_len, n, v.big, extra), lds);
    }
    if constexpr (kSplit) {
        const float strip = lanes_max<kStripLanes>(sum.big);
        if (p.top > 0 && threadIdx.x % kStripLanes == 0)
            strips[(int64_t)blockIdx.x * kStripsPerBlock + threadIdx.x / kStripLanes] = strip;
        if (threadIdx.x == 0) {
            float* q = parts + 3 * (int64_t)blockIdx.x;
            q[0] = v.big, q[1] = v.s, q[2] = v.t;
        }
    } else {
        __shared__ TopScratch top;
        const Values o = row_values(p, v);
        if (threadIdx.x == 0) write_row(p, r, v, o, la, a);
        if (p.top > 0) {
            select_top<T, 1, 1>(p, r, l, mask, v, o, &sum.big, [](int) { return -kInf; }, kBlock, chunk_vecs, chunk_len, top);
        }
    }
}

/* Joins the parts of each row's chunks (at most kBlock of them).  Bound by latency, one block's chain of loads and barriers: one row of 83521
 * with 20 alternatives 8 us, behind 3.3 us of k_policy_chunk. */
template <typename T>
__global__ void __launch_bounds__(kBlock) k_policy_join(const Row p, int chunks, int chunk_vecs, const float* __restrict__ parts,
                                                        const float* __restrict__ strips) {
    __shared__ float lds[3 * (kBlock / 64)];
    __shared__ TopScratch top;
    const int64_t r = blockIdx.x;
    const T* l = static_cast<const T*>(p.logits) + r * p.logits_stride;
    const uint8_t* mask = p.mask ? p.mask + r * p.mask_stride : nullptr;
    const int n_strips = p.top > 0 ? chunks * kStripsPerBlock : 0;
    const float* mine = strips + r * chunks * kStripsPerBlock;
    /* everything the row needs is asked for at once */
    float held[kHold];
    _Pragma("unroll") for (int h = 0; h < kHold; ++h) {
        const int i = held_strip(h, n_strips);
        held[h] = i < n_strips ? mine[i] : -kInf;
    }
    Sum v{-kInf, 0.0f, 0.0f};
    if ((int)threadIdx.x < chunks) {
        const float* q = parts + 3 * (r * chunks + threadIdx.x);
        v = Sum{q[0], q[1], q[2]};
    }
    const int64_t a = row_action(p, r);
    const float la = action_logit<T>(p, l, mask, a);
    v = team_merge<kBlock>(p, v, lds);
    const Values o = row_values(p, v);
    if (threadIdx.x == 0) write_row(p, r, v, o, la, a);
    if (p.top > 0)
        select_top<T, kStripLanes, kHold>(p, r, l, mask, v, o, held, [&](int i) { return mine[i]; }, n_strips, chunk_vecs,
                      (uint32_t)chunk_vecs * kBlock * Kind<T>::kPer, top);
}

/* Gradient of one vector of a plain row, without the action's own part.  The product is the one in which 0 times anything is 0: an
 * exponential of 0 comes with an exponent of -inf where the logit is -inf. */
template <typename T>
__device__ __forceinline__ w4 slope_vec(const Row& p, const Slope& q, const w4& x) {
    constexpr int kPer = Kind<T>::kPer;
    float y[kPer];
    _Pragma("unroll") for (int j = 0; j < kPer; ++j) {
        const float d = fmaf(p.c, Kind<T>::get(x, j), -q.m);
        y[j] = mul_zero_wins(__builtin_amdgcn_exp2f(d), fmaf(q.slope, d, q.base));
    }
    return Kind<T>::pack(y);
}
/* the elements of a cut vector that the row has */
template <typename T>
__device__ __forceinline__ void store_part(T* __restrict__ g, uint32_t i, uint32_t n, const w4& v) {
    _Pragma("unroll") for (int j = 0; j < Kind<T>::kPer - 1; ++j)
        if (i + j < n) {
            const uint32_t bits = sizeof(T) == 4 ? v[j & 3] : v[(j >> 1) & 3] >> (16 * (j & 1));
            __builtin_memcpy(g + i + j, &bits, sizeof(T));
        }
}
/* elements [from, to) of a row one by one: rows that are not plain, and the last few of those that are */
template <typename T, int kTeam>
__device__ void slope_slowly(const Row& p, const Slope& q, const T* l, const uint8_t* mask, T* out, uint32_t from, uint32_t to,
                                          uint32_t action) {
    for (uint32_t i = from + threadIdx.x % kTeam; i < to; i += kTeam) {
        const float x = mask && !mask[i] ? -kInf : Kind<T>::load(l + i);
        float y = 0.0f;
        if (!q.empty && x != -kInf) {
            y = slope_at(p, q, x);
            if (i == action) y += q.at_action;
        }
        Kind<T>::store(out + i, y);
    }
}
/* the action's element, over what its vector's store put there: by the same thread, behind it */
template <typename T>
__device__ __forceinline__ void store_action(const Row& p, const Slope& q, float la, T* out, uint32_t action) {
    if (la != -kInf) Kind<T>::store(out + action, slope_at(p, q, la) + q.at_action);
}

/* Gradient of chunks from the rows' stored statistics; kSlopeGroups groups of vectors a thread, each on its way while the one before it is
 * worked on, the first while the row's statistics come.  1280 x 59049 fp16: 48.8 us with four groups, 52.8 with two, 54.6 with
 * one, which few rows get for the sake of more blocks.  kStream: past the caches, for gradients that do not fit the 256 MiB last-level cache
 * beside the logits, which the forward pass left there: forward and gradient of the same 1280 rows 96 -> 86 us. */
template <typename T, int kSlopeGroups, bool kStream>
__global__ void __launch_bounds__(kBlock) k_policy_slope(const Row p, int chunks) {
    constexpr int kPer = Kind<T>::kPer;
    constexpr uint32_t kStride = kBlock * kPer, kLen = kSlopeGroups * kAhead * kStride;
    const int64_t r = blockIdx.x / chunks;
    const int chunk = blockIdx.x % chunks;
    const T* l = static_cast<const T*>(p.logits) + r * p.logits_stride;
    const uint8_t* mask = p.mask ? p.mask + r * p.mask_stride : nullptr;
    T* out = static_cast<T*>(p.grad_logits) + r * p.grad_stride;
    const uint32_t n = (uint32_t)p.n, skew = skew_of(l), whole = n - (n - skew) % kPer;
    const uint32_t first = skew + (uint32_t)chunk * kLen, end = first + kLen, from = first + threadIdx.x * kPer;
    w4 x[2][kAhead];
    load_raw<T, kAhead>(l, from, kStride, n, x[0]);
    const int64_t a = row_action(p, r);
    const float la = action_logit<T>(p, l, mask, a);
    const Sum v{p.row_stats[2 * r], p.row_stats[2 * r + 1], 0.0f};
    const Slope q = row_slope(p, r, a, v, p.entropy[r], log2f(v.s));
    const uint32_t action = a >= 0 && a < p.n ? (uint32_t)a : ~0u;
    if (!is_plain(p, q)) {
        slope_slowly<T, kBlock>(p, q, l, mask, out, chunk ? first : 0, min(end, n), action);
        return;
    }
    _Pragma("unroll") for (int g = 0; g < kSlopeGroups; ++g) {
        const uint32_t i = from + g * kAhead * kStride;
        if (g + 1 < kSlopeGroups) load_raw<T, kAhead>(l, i + kAhead * kStride, kStride, n, x[(g + 1) & 1]);
        dress<T, kAhead>(mask, i, kStride, n, x[g & 1]);
        _Pragma("unroll") for (int u = 0; u < kAhead; ++u) {
            const uint32_t at = i + u * kStride;
            if (at < whole) store_vec<T, kStream>(out, at, slope_vec<T>(p, q, x[g & 1][u]));
        }
    }
    if (whole >= first && whole < end) slope_slowly<T, kBlock>(p, q, l, mask, out, whole, n, action);
    if (chunk == 0) slope_slowly<T, kBlock>(p, q, l, mask, out, 0, skew, action);
    if (action >= first && action < min(end, whole) && (action - first) / kPer % kBlock == threadIdx.x) store_action<T>(p, q, la, out, action);
}

/* A row that its team holds in registers (V 16-byte vectors a thread): one read, and with kGrad one write, of memory.  Narrow rows share a
 * wave (2 to 4 vectors a thread: what a row costs once — logarithms, outputs — is then spread over several rows); a wave takes
 * rows of up to 16 vectors a thread; a block of 512 threads wider ones, two blocks to a CU (at most 128 registers a thread), one
 * block a row: blocks that start when others end keep loads, sums and stores of different rows in flight, where blocks that walk the rows
 * in step (two a CU, loading the next row into the registers just stored) took 292 us instead of 269 for 4096 x 81920 bf16.
 * kTop: alternatives too, from keys beside the row (Rank), so rows of at most kRankMost logits; 80000 x 1000 bf16 with the five best 84 us,
 * 62 for 40000 x 1000 fp32, where a maximum of 64-bit keys through shared memory took 214 and 73. */
template <typename T, int kTeam, int V, bool kGrad, bool kTop = false>
__global__ void __launch_bounds__(kTeam <= 64 ? kBlock : kTeam, kTeam <= 64 ? 1 : 4) k_policy_row(const Row p) {
    constexpr int kPer = Kind<T>::kPer;
    constexpr uint32_t kStride = kTeam * kPer;
    constexpr int kGroups = V / kAhead, kRest = V % kAhead;
    __shared__ float lds[kTeam <= 64 ? 1 : 3 * (kTeam / 64)];
    const int64_t r = kTeam < 64    ? (int64_t)blockIdx.x * (kBlock / kTeam) + threadIdx.x / kTeam
                      : kTeam == 64 ? (int64_t)blockIdx.x * (kBlock / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)
                                    : blockIdx.x;
    if (r >= p.rows) return; /* a whole team, and nothing below reaches past a team */
    const T* l = static_cast<const T*>(p.logits) + r * p.logits_stride;
    const uint8_t* mask = p.mask ? p.mask + r * p.mask_stride : nullptr;
    const uint32_t n = (uint32_t)p.n, lane = threadIdx.x % kTeam, skew = kTeam > 64 ? skew_of(l) : 0u;
    uint32_t from = skew + lane * kPer;
    w4 x[V];
    load_raw<T, V>(l, from, kStride, n, x);
    const int64_t a = row_action(p, r);
    const float la = action_logit<T>(p, l, mask, a); /* before the gradient may overwrite it */
    const float extra = skew && lane == 0 ? action_logit<T>(p, l, mask, 0) : -kInf;
    Running sum = running_start();
    _Pragma("unroll") for (int j = 0; j < kGroups; ++j) {
        dress<T, kAhead>(mask, from + j * kAhead * kStride, kStride, n, x + j * kAhead);
        take_vecs<T, kAhead>(p, x + j * kAhead, sum);
    }
    if constexpr (kRest != 0) {
        dress<T, kRest>(mask, from + kGroups * kAhead * kStride, kStride, n, x + kGroups * kAhead);
        take_vecs<T, kRest>(p, x + kGroups * kAhead, sum);
    }
    if (skew && lane == 0) take_one(p, extra, sum);
    Sum v = team_merge<kTeam>(p, running_end(p, sum), lds);
    if (is_huge(p, v.big) && fabsf(v.big) < kInf) {
        if (kTeam > 64) __syncthreads();
        v = team_merge<kTeam>(p, sum_slowly<T>(p, l, mask, from, kStride, n, n, v.big, extra), lds);
    }
    const Values o = row_values(p, v);
    if (lane == 0 && p.values) write_row(p, r, v, o, la, a);
    if constexpr (kTop) {
        typename Rank<T>::Key key[V * kPer];
        _Pragma("unroll") for (int j = 0; j < V; ++j)
            _Pragma("unroll") for (int i = 0; i < kPer; ++i)
                key[j * kPer + i] = Rank<T>::make(Kind<T>::get(x[j], i), lane * kPer + j * kStride + i);
        write_best<T, kTeam, V * kPer>(p, r, (int)lane, key, v, o);
    }
    if constexpr (kGrad) {
        const Slope q = row_slope(p, r, a, v, o.entropy, o.log2_s);
        T* out = static_cast<T*>(p.grad_logits) + r * p.grad_stride;
        const uint32_t action = a >= 0 && a < p.n ? (uint32_t)a : ~0u, whole = n - (n - skew) % kPer;
        if (!is_plain(p, q)) {
            slope_slowly<T, kTeam>(p, q, l, mask, out, 0, n, action);
            return;
        }
        asm volatile("" : "+v"(from)); /* the places are worked out anew, not kept since the loads */
        _Pragma("unroll") for (int j = 0; j < V; ++j) {
            const uint32_t i = from + j * kStride;
            unpack_here(x[j]);
            if (i < whole) store_vec<T>(out, i, slope_vec<T>(p, q, x[j]));
            else if (kTeam < 64 && i < n) store_part<T>(out, i, n, slope_vec<T>(p, q, x[j]));
        }
        const uint32_t end = kTeam < 64 ? n : whole;
        if (kTeam >= 64) slope_slowly<T, kTeam>(p, q, l, mask, out, whole, n, action);
        if (skew && lane == 0)
            Kind<T>::store(out, extra == -kInf ? 0.0f : slope_at(p, q, extra) + (action == 0 ? q.at_action : 0.0f));
        if (action >= skew && action < end && (action - skew) / kPer % kTeam == lane) store_action<T>(p, q, la, out, action);
    }
}

int check(const mzs_policy_args* a, bool forward, bool grad) {
    if (!a) return set_error(MZS_E_ARG, "null arguments");
    if (a->dtype < MZS_DTYPE_FLOAT || a->dtype > MZS_DTYPE_HALF) return set_error(MZS_E_ARG, "logits: fp32, bf16 or fp16");
    if (a->rows < 0 || a->n_actions < 1 || a->n_actions > (1 << 28)) return set_error(MZS_E_ARG, "rows >= 0 and 1 <= n_actions <= 2^28");
    if (a->top < 0 || a->top > MZS_POLICY_MAX_TOP) return set_error(MZS_E_ARG, "top: 0 .. MZS_POLICY_MAX_TOP");
    if (!(a->inverse_temperature > 0.0f) || a->inverse_temperature > 1e30f) return set_error(MZS_E_ARG, "inverse_temperature must be positive and finite");
    if (a->logits_stride < 0 || a->mask_stride < 0) return set_error(MZS_E_ARG, "negative row stride");
    if (a->action && a->action_bytes != 4 && a->action_bytes != 8) return set_error(MZS_E_ARG, "actions: int32 or int64");
    if (a->rows == 0) return MZS_OK;
    if (!a->logits || !a->entropy || !a->row_stats) return set_error(MZS_E_ARG, "null buffer");
    if (forward && (!a->log_prob || !a->log_z || (a->top > 0 && (!a->top_log_prob || !a->top_action))))
        return set_error(MZS_E_ARG, "null output");
    if (grad) {
        if (!a->grad_logits) return set_error(MZS_E_ARG, "null gradient");
        if (a->rows > 1 && a->grad_stride < a->n_actions) return set_error(MZS_E_ARG, "gradient rows overlap: grad_stride < n_actions");
        if (a->grad_logits == a->logits && a->rows > 1 && a->grad_stride != a->logits_stride)
            return set_error(MZS_E_ARG, "a gradient in place of the logits needs their stride");
    }
    return MZS_OK;
}

Row pack(const mzs_policy_args& a) {
    Row p;
    p.logits = a.logits, p.mask = a.mask, p.action = a.action;
    p.log_prob = a.log_prob, p.entropy = a.entropy, p.log_z = a.log_z, p.row_stats = a.row_stats;
    p.top_log_prob = a.top_log_prob, p.top_action = a.top_action;
    p.grad_log_prob = a.grad_log_prob, p.grad_entropy = a.grad_entropy, p.grad_log_z = a.grad_log_z;
    p.grad_logits = a.grad_logits;
    p.rows = a.rows, p.n = a.n_actions;
    p.logits_stride = a.logits_stride, p.mask_stride = a.mask_stride, p.grad_stride = a.grad_stride;
    p.action_bytes = a.action_bytes, p.top = a.top;
    p.scale = a.inverse_temperature, p.values = 1;
    p.c = (float)((double)a.inverse_temperature * kLog2e);
    return p;
}

/* widest row whose gradient sums the row again in registers rather than read its statistics back */
constexpr int64_t kRegainMost = 2048;

template <typename T, bool kForward, bool kGrad, bool kTop>
void launch_lanes(const Row& p, hipStream_t st) {
    const int64_t blocks = (p.rows + kBlock - 1) / kBlock;
    const dim3 grid((unsigned)(blocks < 65536 ? blocks : 65536));
    if (p.n <= 4) hipLaunchKernelGGL((k_policy_lanes<T, 4, kForward, kGrad, kTop>), grid, dim3(kBlock), 0, st, p);
    else hipLaunchKernelGGL((k_policy_lanes<T, 8, kForward, kGrad, kTop>), grid, dim3(kBlock), 0, st, p);
}

template <typename T>
void launch_forward(const Row& p, const PolicyCut& c, void* workspace, hipStream_t st) {
    if (c.chunks == 1) {
        hipLaunchKernelGGL((k_policy_chunk<T, false>), dim3((unsigned)p.rows), dim3(kBlock), 0, st, p, 1, c.vecs, nullptr, nullptr);
        return;
    }
    float* parts = static_cast<float*>(workspace);
    float* strips = parts + 3 * p.rows * c.chunks;
    hipLaunchKernelGGL((k_policy_chunk<T, true>), dim3((unsigned)(p.rows * c.chunks)), dim3(kBlock), 0, st, p, c.chunks, c.vecs, parts, strips);
    hipLaunchKernelGGL(k_policy_join<T>, dim3((unsigned)p.rows), dim3(kBlock), 0, st, p, c.chunks, c.vecs, (const float*)parts,
                       (const float*)strips);
}
template <typename T>
void launch_slope(const Row& p, hipStream_t st) {
    const int64_t group = (int64_t)kAhead * kBlock * Kind<T>::kPer, groups = (p.n + group - 1) / group;
    if (p.rows * groups < 4096) {
        hipLaunchKernelGGL((k_policy_slope<T, 1, false>), dim3((unsigned)(p.rows * groups)), dim3(kBlock), 0, st, p, (int)groups);
    } else {
        const int chunks = (int)((groups + 3) / 4);
        const bool stream = 2 * p.rows * p.n * (int64_t)sizeof(T) > ((int64_t)256 << 20);
        hipLaunchKernelGGL((stream ? k_policy_slope<T, 4, true> : k_policy_slope<T, 4, false>), dim3((unsigned)(p.rows * chunks)), dim3(kBlock), 0,
                           st, p, chunks);
    }
}

/* rows in registers: up to kPolicyWaveVecs vectors a lane of a wave, kRowVecs a thread of a block of kRowThreads */
constexpr int kRowThreads = 512, kRowVecs = 24;
template <typename T>
bool fits_block(int64_t n) { return n <= (int64_t)kRowThreads * kRowVecs * Kind<T>::kPer; }
template <typename T, bool kGrad>
void launch_wave_row(const Row& p, hipStream_t st) {
    const int64_t all = (p.n + Kind<T>::kPer - 1) / Kind<T>::kPer;
    const auto go = [&](auto kernel, int team) {
        const int64_t per_block = kBlock / team;
        hipLaunchKernelGGL(kernel, dim3((unsigned)((p.rows + per_block - 1) / per_block)), dim3(kBlock), 0, st, p);
    };
    if (all <= 2) go(k_policy_row<T, 1, 2, kGrad>, 1);
    else if (all <= 4) go(k_policy_row<T, 2, 2, kGrad>, 2);
    else if (all <= 8) go(k_policy_row<T, 4, 2, kGrad>, 4);
    else if (all <= 12) go(k_policy_row<T, 4, 3, kGrad>, 4);
    else if (all <= 16) go(k_policy_row<T, 4, 4, kGrad>, 4);
    else if (all <= 24) go(k_policy_row<T, 8, 3, kGrad>, 8);
    else if (all <= 32) go(k_policy_row<T, 8, 4, kGrad>, 8);
    else if (all <= 48) go(k_policy_row<T, 16, 3, kGrad>, 16);
    else if (all <= 64) go(k_policy_row<T, 16, 4, kGrad>, 16);
    else if (all <= 96) go(k_policy_row<T, 32, 3, kGrad>, 32);
    else if (all <= 128) go(k_policy_row<T, 32, 4, kGrad>, 32);
    else if (all <= 192) go(k_policy_row<T, 64, 3, kGrad>, 64);
    else if (all <= 256) go(k_policy_row<T, 64, 4, kGrad>, 64);
    else if (all <= 384) go(k_policy_row<T, 64, 6, kGrad>, 64);
    else if (all <= 512) go(k_policy_row<T, 64, 8, kGrad>, 64);
    else if (all <= 768) go(k_policy_row<T, 64, 12, kGrad>, 64);
    else go(k_policy_row<T, 64, 16, kGrad>, 64);
}
/* With alternatives, up to kRankMost logits: few lanes a row, as each choice costs its team's butterfly and then little for a row of
 * 12 to 24 logits a lane - unless the rows are so few that their lanes do not fill the card, where more of them end sooner. */
template <typename T>
void launch_wave_top(const Row& p, hipStream_t st) {
    constexpr int V = sizeof(T) == 4 ? 4 : 2, W = 3; /* fp32: 3 or 4 vectors a lane; 2-byte types: 2 or 3 */
    constexpr int kSmall = V < W ? V : W, kLarge = V < W ? W : V;
    const int64_t all = (p.n + Kind<T>::kPer - 1) / Kind<T>::kPer;
    const auto go = [&](auto kernel, int team) {
        const int64_t per_block = kBlock / team;
        hipLaunchKernelGGL(kernel, dim3((unsigned)((p.rows + per_block - 1) / per_block)), dim3(kBlock), 0, st, p);
    };
    if (p.rows * all <= 64 * 2048 && all <= 64) {
        if (all <= 4) go(k_policy_row<T, 4, 1, false, true>, 4);
        else if (all <= 8) go(k_policy_row<T, 8, 1, false, true>, 8);
        else if (all <= 16) go(k_policy_row<T, 16, 1, false, true>, 16);
        else if (all <= 32) go(k_policy_row<T, 32, 1, false, true>, 32);
        else go(k_policy_row<T, 64, 1, false, true>, 64);
    } else if (all <= kSmall) go(k_policy_row<T, 1, kSmall, false, true>, 1);
    else if (all <= kLarge) go(k_policy_row<T, 1, kLarge, false, true>, 1);
    else if (all <= 2 * kSmall) go(k_policy_row<T, 2, kSmall, false, true>, 2);
    else if (all <= 2 * kLarge) go(k_policy_row<T, 2, kLarge, false, true>, 2);
    else if (all <= 4 * kSmall) go(k_policy_row<T, 4, kSmall, false, true>, 4);
    else if (all <= 4 * kLarge) go(k_policy_row<T, 4, kLarge, false, true>, 4);
    else if (all <= 8 * kSmall) go(k_policy_row<T, 8, kSmall, false, true>, 8);
    else if (all <= 8 * kLarge) go(k_policy_row<T, 8, kLarge, false, true>, 8);
    else if (all <= 16 * kSmall) go(k_policy_row<T, 16, kSmall, false, true>, 16);
    else if (all <= 16 * kLarge) go(k_policy_row<T, 16, kLarge, false, true>, 16);
    else if (all <= 32 * kSmall) go(k_policy_row<T, 32, kSmall, false, true>, 32);
    else if (all <= 32 * kLarge) go(k_policy_row<T, 32, kLarge, false, true>, 32);
    else if (all <= 64 * kSmall) go(k_policy_row<T, 64, kSmall, false, true>, 64);
    else if (all <= 64 * kLarge) go(k_policy_row<T, 64, kLarge, false, true>, 64);
    else if (sizeof(T) == 4 && all <= 64 * 6) go(k_policy_row<T, 64, sizeof(T) == 4 ? 6 : 2 * V, false, true>, 64);
    else go(k_policy_row<T, 64, 2 * V, false, true>, 64);
}
/* Vectors a thread: up to 16 the steps are wide, as places that stay empty cost little (a row of 9 in 12 places 265 us, in 10 266; of 13 in
 * 16 262, in 14 267; 3.4e8 bf16 logits in all).  Beyond, 2-byte types run out of registers and their steps are narrow: rows of 17 take 279 in 20
 * places, 296 in 22 and 315 in 24, of 19 268, 275 and 309, of 21.7 285 in 22 and 307 in 24; of 17 in 18 places 275, not worth an instance more.
 * Fp32 takes the same time in 24 places as in any (within 1 %, 17 to 23.6 vectors). */
template <typename T>
void launch_block_row(const Row& p, hipStream_t st) {
    const int64_t all = (p.n + (int64_t)kRowThreads * Kind<T>::kPer - 1) / ((int64_t)kRowThreads * Kind<T>::kPer);
    const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)p.rows), dim3(kRowThreads), 0, st, p); };
    constexpr bool kHalf = sizeof(T) == 2;
    if (all <= 3) go(k_policy_row<T, kRowThreads, 3, true>);
    else if (all <= 4) go(k_policy_row<T, kRowThreads, 4, true>);
    else if (all <= 6) go(k_policy_row<T, kRowThreads, 6, true>);
    else if (all <= 8) go(k_policy_row<T, kRowThreads, 8, true>);
    else if (all <= 12) go(k_policy_row<T, kRowThreads, 12, true>);
    else if (all <= 16) go(k_policy_row<T, kRowThreads, 16, true>);
    else if (kHalf && all <= 20) go(k_policy_row<T, kRowThreads, kHalf ? 20 : kRowVecs, true>);
    else if (kHalf && all <= 22) go(k_policy_row<T, kRowThreads, kHalf ? 22 : kRowVecs, true>);
    else go(k_policy_row<T, kRowThreads, kRowVecs, true>);
}

/* rows [r, r + rows) of a call */
template <typename T>
Row rows_from(Row p, int64_t r, int64_t rows) {
    const auto on = [r](auto* q, int64_t each) { return q ? q + r * each : q; };
    p.logits = on(static_cast<const T*>(p.logits), p.logits_stride);
    p.mask = on(p.mask, p.mask_stride);
    p.action = on(static_cast<const uint8_t*>(p.action), p.action_bytes);
    p.log_prob = on(p.log_prob, 1), p.entropy = on(p.entropy, 1), p.log_z = on(p.log_z, 1), p.row_stats = on(p.row_stats, 2);
    p.top_log_prob = on(p.top_log_prob, p.top), p.top_action = on(p.top_action, p.top);
    p.grad_log_prob = on(p.grad_log_prob, 1), p.grad_entropy = on(p.grad_entropy, 1), p.grad_log_z = on(p.grad_log_z, 1);
    p.grad_logits = on(static_cast<T*>(p.grad_logits), p.grad_stride);
    p.rows = rows;
    return p;
}
/* The ways, by the width of the row (and how a call needs it):
 *   up to 8 logits              a lane a row, a logit at a time                             k_policy_lanes
 *   up to 16 vectors a lane     a row in a team's registers; with alternatives up to 2048   k_policy_row, teams up to a wave
 *   up to 24 vectors a thread   forward and gradient of a row in a block's registers        k_policy_row, a block
 *   beyond                      chunks and their join; the gradient from the statistics     k_policy_chunk, k_policy_join, k_policy_slope */
template <typename T>
void run_kind(const Row& all, const PolicyPlan& plan, void* workspace, hipStream_t st, bool forward, bool grad) {
    const bool lanes = all.n <= kPolicyLanesMost, wave = !lanes && policy_fits_wave(all.n, Kind<T>::kPer);
    const bool both = forward && grad && all.top == 0;
    policy_launches(all.rows, plan, [&](int64_t first, int64_t rows, const PolicyPlan&) {
        const Row p = rows_from<T>(all, first, rows);
        if (both && wave) {
            launch_wave_row<T, true>(p, st);
            return;
        }
        if (both && lanes) {
            launch_lanes<T, true, true, false>(p, st);
            return;
        }
        if (both && fits_block<T>(p.n)) {
            launch_block_row<T>(p, st);
            return;
        }
        if (forward) {
            if (wave && p.top == 0) launch_wave_row<T, false>(p, st);
            else if (wave && p.n <= kRankMost) launch_wave_top<T>(p, st);
            else if (lanes && p.top > 0) launch_lanes<T, true, false, true>(p, st);
            else if (lanes) launch_lanes<T, true, false, false>(p, st);
            else launch_forward<T>(p, plan.cut, workspace, st);
        }
        if (grad) {
            Row g = p;
            g.values = 0;
            if (wave && p.n <= kRegainMost) launch_wave_row<T, true>(g, st);
            else if (lanes) launch_lanes<T, false, true, false>(p, st);
            else launch_slope<T>(p, st);
        }
    });
}

PolicyPlan plan_of(const mzs_policy_args& a) { return policy_plan(a.rows, a.n_actions, a.dtype == MZS_DTYPE_FLOAT ? 4 : 8, a.top); }

int run(const mzs_policy_args* a, void* stream, bool forward, bool grad) {
    const int rc = check(a, forward, grad);
    if (rc || a->rows == 0) return rc;
    const PolicyPlan plan = plan_of(*a);
    if (forward && plan.workspace && (!a->workspace || a->workspace_bytes < plan.workspace))
        return set_error(MZS_E_ARG, "workspace too small (mzs_policy_workspace)");
    DeviceScope scope(a->device);
    if (scope.status != hipSuccess) return hip_error("mzs_policy: device", scope.status);
    const Row p = pack(*a);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (a->dtype == MZS_DTYPE_FLOAT) run_kind<float>(p, plan, a->workspace, st, forward, grad);
    else if (a->dtype == MZS_DTYPE_BFLOAT) run_kind<__bf16>(p, plan, a->workspace, st, forward, grad);
    else run_kind<_Float16>(p, plan, a->workspace, st, forward, grad);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MZS_OK : hip_error("mzs_policy: launch", e);
}

}  // namespace
}  // namespace mzs

extern "C" {

int mzs_policy_workspace(const mzs_policy_args* args, size_t* bytes_out) {
    if (!args || !bytes_out) return mzs::set_error(MZS_E_ARG, "null argument");
    if (args->dtype < MZS_DTYPE_FLOAT || args->dtype > MZS_DTYPE_HALF || args->rows < 0 || args->n_actions < 1 || args->n_actions > (1 << 28))
        return mzs::set_error(MZS_E_ARG, "fp32, bf16 or fp16; rows >= 0 and 1 <= n_actions <= 2^28");
    *bytes_out = args->rows ? mzs::plan_of(*args).workspace : 0;
    return MZS_OK;
}
int mzs_policy_log_probs(const mzs_policy_args* args, void* stream) { return mzs::run(args, stream, true, false); }
int mzs_policy_log_probs_grad(const mzs_policy_args* args, void* stream) { return mzs::run(args, stream, false, true); }
int mzs_policy_log_probs_train(const mzs_policy_args* args, void* stream) { return mzs::run(args, stream, true, true); }

}  // extern "C"
