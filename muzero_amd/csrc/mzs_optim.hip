/*
 * mzs_optim.hip — global gradient norm and AdamW step over many tensors (include/mzsearch.h, mzs_optim_*, mzs_grad_norm,
 * mzs_adamw_step).
 *
 * Mathematics.  norm = |scale| sqrt(sum g^2), in fp64 from the first product on, in a fixed order.  A step t with clip = min(1, max_norm /
 * (norm + 1e-6)), g' = grad_scale clip g:  m = b1 m + (1 - b1) g', v = b2 v + (1 - b2) g'^2, w = w (1 - lr wd) - lr / (1 - b1^t) m /
 * (sqrt(v) / sqrt(1 - b2^t) + eps), all in fp32.  8-bit states hold m and sqrt(v) as e4m3 codes under one power of two for each 32
 * elements, rounded up with the probability of the remainder.
 *
 * Work is cut into tiles of kTile elements of one tensor; a table in device memory says which tensor a tile is of.  All of it is bound by
 * memory but for short lists, which launches bound, and 2-byte weights with 8-bit states, which the codes' arithmetic bounds.
 */
#include "mzs_error.h"

#include <cmath>
#include <cstddef>
#include <cstdint>
#include <cstring>

namespace mzs {
namespace {

constexpr int kBlock = 256;
constexpr int kTile = 4096;       /* elements of a tile */
constexpr int kFillEntries = 120; /* table entries a launch carries in its arguments */
constexpr int kMaxPartials = 2048; /* 8 blocks on each of 256 CUs */
constexpr int kVec = 4;           /* elements a thread takes at once */
constexpr int kSmallTiles = 16;   /* most tiles of k_adamw_small: one to a wave of its blocks */
constexpr int kSmallBlock = 64 * kSmallTiles;
static_assert(kSmallBlock * kVec == kTile, "a block of k_adamw_small updates a tile at once");
constexpr int kGroup = MZS_OPTIM_BLOCK;

struct Entry {
    void* data; /* null: no tensor */
    int64_t count, first_tile, state_at;
};
static_assert(sizeof(Entry) == MZS_OPTIM_ENTRY_BYTES, "entry size");

struct FillArgs {
    Entry entries[kFillEntries];
};

__global__ void __launch_bounds__(128) k_optim_table(const FillArgs a, Entry* __restrict__ table, int at, int n) {
    if ((int)threadIdx.x < n) table[at + threadIdx.x] = a.entries[threadIdx.x];
}

struct bf16 {
    uint16_t bits;
};
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(bf16 v) { return __uint_as_float((uint32_t)v.bits << 16); }
__device__ __forceinline__ float to_float(_Float16 v) { return (float)v; }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ uint32_t bf16_bits(float v) { /* nearest even; a NaN stays one */
    const uint32_t b = __float_as_uint(v);
    return v != v ? 0x7fc0u : (b + 0x7fffu + ((b >> 16) & 1u)) >> 16;
}
__device__ __forceinline__ void put(bf16* p, float v) { p->bits = (uint16_t)bf16_bits(v); }
__device__ __forceinline__ void put(_Float16* p, float v) { *p = (_Float16)v; }

/* four (or eight) consecutive elements in one access; tensors may start at any element, which costs the hardware nothing from 4 bytes on */
typedef uint32_t w2 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t w4 __attribute__((ext_vector_type(4), aligned(2)));
typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ float low_half(uint32_t v, bf16) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float high_half(uint32_t v, bf16) { return __uint_as_float(v & 0xffff0000u); }
__device__ __forceinline__ float low_half(uint32_t v, _Float16) { return (float)__builtin_bit_cast(h2, v).x; }
__device__ __forceinline__ float high_half(uint32_t v, _Float16) { return (float)__builtin_bit_cast(h2, v).y; }
__device__ __forceinline__ uint32_t pack_halves(float a, float b, bf16) { return bf16_bits(a) | (bf16_bits(b) << 16); }
__device__ __forceinline__ uint32_t pack_halves(float a, float b, _Float16) {
    return __builtin_bit_cast(uint32_t, h2{(_Float16)a, (_Float16)b});
}
template <typename T>
struct Quad { /* as it comes from memory */
    w2 raw;
    template <bool kStream>
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (kStream) raw = __builtin_nontemporal_load(reinterpret_cast<const w2*>(p));
        else raw = *reinterpret_cast<const w2*>(p);
    }
    __device__ __forceinline__ float get(int j) const {
        const uint32_t v = j < 2 ? raw.x : raw.y;
        return j & 1 ? high_half(v, T()) : low_half(v, T());
    }
    template <bool kStream>
    static __device__ __forceinline__ void store(T* p, const float* v) {
        const w2 x{pack_halves(v[0], v[1], T()), pack_halves(v[2], v[3], T())};
        if constexpr (kStream) __builtin_nontemporal_store(x, reinterpret_cast<w2*>(p));
        else *reinterpret_cast<w2*>(p) = x;
    }
};
template <>
struct Quad<float> {
    f4 raw;
    template <bool kStream>
    __device__ __forceinline__ void load(const float* p) {
        if constexpr (kStream) raw = __builtin_nontemporal_load(reinterpret_cast<const f4*>(p));
        else raw = *reinterpret_cast<const f4*>(p);
    }
    __device__ __forceinline__ float get(int j) const { return raw[j]; }
    template <bool kStream>
    static __device__ __forceinline__ void store(float* p, const float* v) {
        const f4 x{v[0], v[1], v[2], v[3]};
        if constexpr (kStream) __builtin_nontemporal_store(x, reinterpret_cast<f4*>(p));
        else *reinterpret_cast<f4*>(p) = x;
    }
};

/* The tensor that tile `tile` is of: the last entry with first_tile <= tile (empty tensors have no tiles).  The lanes of a wave look at
 * 64 entries at once: two dependent loads for 4096 tensors instead of twelve. */
__device__ __forceinline__ int find_tensor(const Entry* __restrict__ table, int n, int64_t tile) {
    const int lane = threadIdx.x & 63;
    int lo = 0, len = n;
    while (len > 1) {
        const int s = (len + 63) >> 6;
        const int at = lane * s;
        const bool before = at < len && table[lo + at].first_tile <= tile;
        const int hit = __popcll(__ballot(before)) - 1; /* lane 0's entry is always one */
        lo += hit * s;
        len = len - hit * s < s ? len - hit * s : s;
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

/* fixed-order sum over the block; the total in thread 0 */
__device__ __forceinline__ double block_sum(double v, double* lds) {
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    double sum = 0.0;
    for (int w = 0; w < kBlock / 64; ++w) sum += lds[w];
    return sum;
}

/* squares of elements [from, to) of one tensor, this thread's share, in fp64 (fp32 squares overflow from 1.8e19 on and vanish
 * below 1e-23; the fp64 fma runs at the fp32 rate here, so the loads bound it either way) */
template <typename G, bool kStream>
__device__ __forceinline__ double sum_squares(const G* __restrict__ g, int64_t from, int64_t to, int thread, int threads) {
    constexpr int kUnroll = 2; /* 300M bf16: 107 us; 117 with four, 123 with eight: more waves do more than more loads each */
    constexpr int kWide = sizeof(G) == 4 ? 4 : 8; /* 16 bytes */
    double sum[2] = {0.0, 0.0};
    int64_t i = from + (int64_t)thread * kWide;
    const int64_t step = (int64_t)threads * kWide;
    for (; i + (kUnroll - 1) * step + kWide <= to; i += kUnroll * step) {
        Quad<G> q[kUnroll][kWide / 4];
        _Pragma("unroll") for (int u = 0; u < kUnroll; ++u) {
            if constexpr (kWide == 4) {
                q[u][0].template load<kStream>(g + i + u * step);
            } else {
                const w4* at = reinterpret_cast<const w4*>(g + i + u * step);
                w4 raw;
                if constexpr (kStream) raw = __builtin_nontemporal_load(at);
                else raw = *at;
                q[u][0].raw = w2{raw.x, raw.y}, q[u][1].raw = w2{raw.z, raw.w};
            }
        }
        _Pragma("unroll") for (int u = 0; u < kUnroll; ++u)
            _Pragma("unroll") for (int j = 0; j < kWide; ++j) {
                const double x = (double)q[u][j / 4].get(j % 4);
                sum[j & 1] = fma(x, x, sum[j & 1]);
            }
    }
    for (; i < to; i += step) {
        const int64_t end = i + kWide < to ? i + kWide : to;
        for (int64_t k = i; k < end; ++k) {
            const double x = (double)to_float(g[k]);
            sum[0] = fma(x, x, sum[0]);
        }
    }
    return sum[0] + sum[1];
}

/* One read of everything: a block takes a run of consecutive tiles, which is one contiguous range for each tensor it
 * meets; two 16-byte loads a thread in flight.  kStream: past the caches, for a long
 * list that nothing reads again at once (300M bf16: 94 us instead of 106); in front of an update the gradients are left in the last-level
 * cache for it (100M bf16 with master: 52 + 459 us, 33 + 492 past the caches). */
template <typename G, bool kStream>
__global__ void __launch_bounds__(kBlock) k_norm_partial(const Entry* __restrict__ table, int n, int64_t n_tiles,
                                                         double* __restrict__ partial) {
    __shared__ double lds[kBlock / 64];
    const int64_t per = n_tiles / gridDim.x, more = n_tiles % gridDim.x, b = blockIdx.x;
    int64_t tile = b * per + (b < more ? b : more);
    const int64_t end = tile + per + (b < more ? 1 : 0);
    double sum = 0.0;
    int which = find_tensor(table, n, tile);
    while (tile < end && which < n) {
        const Entry e = table[which];
        const int64_t tiles = (e.count + kTile - 1) / kTile;
        const int64_t last = e.first_tile + tiles < end ? e.first_tile + tiles : end;
        if (e.data && last > tile) {
            const int64_t to = (last - e.first_tile) * kTile;
            sum += sum_squares<G, kStream>(static_cast<const G*>(e.data), (tile - e.first_tile) * kTile, to < e.count ? to : e.count, threadIdx.x,
                               kBlock);
        }
        if (last > tile) tile = last;
        ++which;
    }
    const double total = block_sum(sum, lds);
    if (threadIdx.x == 0) partial[blockIdx.x] = total;
}

struct Control {
    int32_t step, skipped;
    uint32_t ticket;    /* blocks of a running k_adamw_small that have read `step` */
    int32_t skip;       /* this step is skipped               */
    uint32_t key;       /* dither key of this step            */
    float scale;        /* grad_scale * clip                  */
    float step_size;    /* lr / (1 - beta1^t)                 */
    float decay;        /* 1 - lr * weight_decay              */
    float inv_root_2;   /* 1 / sqrt(1 - beta2^t)              */
};
static_assert(sizeof(Control) <= MZS_OPTIM_CONTROL_BYTES && offsetof(Control, skip) == 4 * MZS_OPTIM_CONTROL_SKIP, "control layout");

struct StepArgs {
    const Entry* params;
    const Entry* grads;
    float* master;
    void* m;
    void* v;
    uint8_t* m_exp;
    uint8_t* v_exp;
    Control* control;
    float* norm;
    const float* lr_dev;
    const double* partial;
    int64_t n_tiles;
    double lr, beta1, beta2, weight_decay, max_norm, grad_scale;
    uint64_t seed;
    float b1, one_minus_b1, b2, one_minus_b2, eps;
    int n, n_partial;
};

/* a bijection of 32-bit words: two rounds of shift, exclusive or and an odd multiplier (the fractional bits of sqrt 3 and
 * sqrt 2, which are odd) */
__device__ __forceinline__ uint32_t mix(uint32_t x) {
    x ^= x >> 16;
    x *= 0xBB67AE85u;
    x ^= x >> 15;
    x *= 0x6A09E667u;
    return x ^ (x >> 16);
}

__device__ __forceinline__ double join_partials(const double* partial, int n, double* lds) {
    double sum = 0.0;
    for (int i = threadIdx.x; i < n; i += kBlock) sum += partial[i];
    return block_sum(sum, lds);
}

__global__ void __launch_bounds__(kBlock) k_norm_join(const double* __restrict__ partial, int n, double scale,
                                                      float* __restrict__ norm) {
    __shared__ double lds[kBlock / 64];
    const double total = join_partials(partial, n, lds);
    if (threadIdx.x == 0) norm[0] = (float)(scale * sqrt(total));
}

/* x^t by squaring: a relative error of about t 2^-53, which 1 - x^t does not see */
__device__ __forceinline__ double power(double x, uint32_t t) {
    double y = 1.0;
    for (; t; t >>= 1, x *= x)
        if (t & 1u) y *= x;
    return y;
}
/* what step t needs; false: the step is skipped */
__device__ __forceinline__ bool step_values(const StepArgs& a, float norm, int t, Control& c) {
    c.skip = a.max_norm > 0.0 && !(fabsf(norm) < __builtin_inff());
    if (c.skip) return false;
    const double lr = a.lr_dev ? (double)a.lr_dev[0] : a.lr;
    float clip = 1.0f;
    if (a.max_norm > 0.0) clip = fminf(1.0f, (float)a.max_norm / (norm + 1e-6f));
    c.key = mix((uint32_t)a.seed ^ mix((uint32_t)t * 0x9E3779B9u + (uint32_t)(a.seed >> 32)));
    c.scale = (float)a.grad_scale * clip;
    c.step_size = (float)(lr / (1.0 - power(a.beta1, (uint32_t)t)));
    c.decay = (float)(1.0 - lr * a.weight_decay);
    c.inv_root_2 = (float)(1.0 / sqrt(1.0 - power(a.beta2, (uint32_t)t)));
    return true;
}

/* One block before the update, 4.5 us: the norm (joined from n_partial sums, or given), clipping, bias corrections, the step counter */
__global__ void __launch_bounds__(kBlock) k_adamw_begin(const StepArgs a) {
    __shared__ double lds[kBlock / 64];
    float norm = 0.0f;
    if (a.n_partial > 0) {
        norm = (float)(fabs(a.grad_scale) * sqrt(join_partials(a.partial, a.n_partial, lds)));
        if (threadIdx.x == 0 && a.norm) a.norm[0] = norm;
    } else if (a.max_norm > 0.0) {
        norm = a.norm[0];
    }
    if (threadIdx.x != 0) return;
    Control c;
    const int t = a.control->step + 1;
    if (step_values(a, norm, t, c)) {
        a.control->step = t;
        a.control->key = c.key, a.control->scale = c.scale, a.control->step_size = c.step_size;
        a.control->decay = c.decay, a.control->inv_root_2 = c.inv_root_2;
    } else {
        a.control->skipped += 1;
    }
    a.control->skip = c.skip;
}

/* ---- 8-bit states: e4m3 codes under a shared power of two.  The conversions are the hardware's: its stochastic rounding
 * with the 16 dither bits in the high half of the random word is floor(|y| / step + r / 65536), subnormal codes included. */
__device__ __forceinline__ float exponent_value(uint32_t e) { /* 2^(e - 127); 255: NaN */
    return e == 255u ? __builtin_nanf("") : e ? __uint_as_float(e << 23) : 5.87747175411143754e-39f;
}
/* exponent byte of a block whose largest magnitude has these bits: 448 = 1.75 * 2^8, a mantissa above 1.75 carries */
__device__ __forceinline__ uint32_t block_exponent(uint32_t most) {
    const int e = (int)((most + 0x1fffffu) >> 23) - 8;
    return most >= 0x7f800000u ? 255u : (uint32_t)(e < 0 ? 0 : e);
}
/* largest of a lane's value over its eight neighbours' */
__device__ __forceinline__ uint32_t max_over_8(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, true));  /* quad_perm 1 0 3 2 */
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, true));  /* quad_perm 2 3 0 1 */
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xf, 0xf, true)); /* row_half_mirror: the other four */
    return v;
}

/* y rounded by dither into byte j of `codes` */
__device__ __forceinline__ uint32_t put_code(float y, uint32_t dither, uint32_t codes, int j) {
    return (uint32_t)(j == 0   ? __builtin_amdgcn_cvt_sr_fp8_f32(y, (int)dither, (int)codes, 0)
                      : j == 1 ? __builtin_amdgcn_cvt_sr_fp8_f32(y, (int)dither, (int)codes, 1)
                      : j == 2 ? __builtin_amdgcn_cvt_sr_fp8_f32(y, (int)dither, (int)codes, 2)
                               : __builtin_amdgcn_cvt_sr_fp8_f32(y, (int)dither, (int)codes, 3));
}

__device__ __forceinline__ float adamw(float w, float& m, float& v, float& root, float g, const StepArgs& a, const Control& c) {
    m = m * a.b1 + g * a.one_minus_b1;
    v = v * a.b2 + g * g * a.one_minus_b2;
    root = __builtin_amdgcn_sqrtf(v); /* root and reciprocal to one unit in the last place: the correctly rounded ones take ten times the
                                         operations, which bound the 8-bit step */
    return w * c.decay - c.step_size * (m * __builtin_amdgcn_rcpf(root * c.inv_root_2 + a.eps));
}

/* a quad's loads and stores; kWhole: all four elements exist, else `count` of them do (tail of a tensor) */
template <typename T, bool kWhole, bool kStream>
__device__ __forceinline__ void load_quad(const T* p, int count, float* out) {
    if (kWhole) {
        Quad<T> q;
        q.template load<kStream>(p);
        _Pragma("unroll") for (int j = 0; j < kVec; ++j) out[j] = q.get(j);
    } else {
        _Pragma("unroll") for (int j = 0; j < kVec; ++j) out[j] = j < count ? to_float(p[j]) : 0.0f;
    }
}
template <typename T, bool kWhole, bool kStream>
__device__ __forceinline__ void store_quad(T* p, int count, const float* v) {
    if (kWhole) Quad<T>::template store<kStream>(p, v);
    else _Pragma("unroll") for (int j = 0; j < kVec; ++j) if (j < count) put(p + j, v[j]);
}

/* One tile by kThreads threads: kTile / (kThreads * kVec) quads a thread, every load of them issued before the first is used (two at a time
 * with byte codes: their arithmetic, 57 operations an element, wants more waves rather than more loads; 64M bf16 167 us, 175 with four). */
template <typename P, typename G, bool kBytes, bool kWhole, int kThreads, bool kStream>
__device__ __forceinline__ void step_tile(const StepArgs& a, const Control& c, P* __restrict__ param, const G* __restrict__ grad,
                                          int64_t state_at, int count) {
    constexpr int kStep = kThreads * kVec, kMost = kTile / kStep, kUnroll = !kWhole ? 1 : kBytes && kMost > 2 ? 2 : kMost;
    const bool master = a.master != nullptr;
    for (int i0 = 0; i0 < (kWhole ? kTile : count); i0 += kUnroll * kStep) {
        float g[kUnroll][kVec], w[kUnroll][kVec], m[kUnroll][kVec], v[kUnroll][kVec];
        uint32_t mc[kUnroll], vc[kUnroll], me[kUnroll], ve[kUnroll];
        _Pragma("unroll") for (int u = 0; u < kUnroll; ++u) {
            const int i = i0 + u * kStep + (int)threadIdx.x * kVec, left = count - i;
            const int64_t k = state_at + i;
            load_quad<G, kWhole, kStream>(grad + i, left, g[u]);
            if (master) load_quad<float, kWhole, kStream>(a.master + k, left, w[u]);
            else load_quad<P, kWhole, kStream>(param + i, left, w[u]);
            if (kBytes) { /* codes come in whole blocks: the state is padded, the blocks' zeros behind a tensor stay zeros */
                mc[u] = vc[u] = me[u] = ve[u] = 0;
                if (kWhole || left > 0) {
                    mc[u] = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.m) + k);
                    vc[u] = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.v) + k);
                    me[u] = a.m_exp[k / kGroup], ve[u] = a.v_exp[k / kGroup];
                }
            } else {
                load_quad<float, kWhole, kStream>(static_cast<const float*>(a.m) + k, left, m[u]);
                load_quad<float, kWhole, kStream>(static_cast<const float*>(a.v) + k, left, v[u]);
            }
        }
        _Pragma("unroll") for (int u = 0; u < kUnroll; ++u) {
            const int i = i0 + u * kStep + (int)threadIdx.x * kVec, left = count - i;
            const int64_t k = state_at + i;
            float root[kVec];
            if (kBytes) {
                const float sm = exponent_value(me[u]), sv = exponent_value(ve[u]);
                const auto m01 = __builtin_amdgcn_cvt_pk_f32_fp8((int)mc[u], false), m23 = __builtin_amdgcn_cvt_pk_f32_fp8((int)mc[u], true);
                const auto v01 = __builtin_amdgcn_cvt_pk_f32_fp8((int)vc[u], false), v23 = __builtin_amdgcn_cvt_pk_f32_fp8((int)vc[u], true);
                m[u][0] = m01[0] * sm, m[u][1] = m01[1] * sm, m[u][2] = m23[0] * sm, m[u][3] = m23[1] * sm;
                const float r[kVec] = {v01[0] * sv, v01[1] * sv, v23[0] * sv, v23[1] * sv};
                _Pragma("unroll") for (int j = 0; j < kVec; ++j) v[u][j] = r[j] * r[j];
            }
            _Pragma("unroll") for (int j = 0; j < kVec; ++j)
                w[u][j] = adamw(w[u][j], m[u][j], v[u][j], root[j], g[u][j] * c.scale, a, c);
            if (kBytes) {
                uint32_t most_m = 0, most_v = 0; /* as bits, so that a NaN is the largest */
                _Pragma("unroll") for (int j = 0; j < kVec; ++j) if (kWhole || j < left) {
                    most_m = max(most_m, __float_as_uint(m[u][j]) & 0x7fffffffu);
                    most_v = max(most_v, __float_as_uint(root[j]) & 0x7fffffffu);
                }
                me[u] = block_exponent(max_over_8(most_m)), ve[u] = block_exponent(max_over_8(most_v));
                const float sm = __uint_as_float((254u - me[u]) << 23), sv = __uint_as_float((254u - ve[u]) << 23);
                const uint32_t x = (uint32_t)k * 0x9E3779B1u + c.key;
                mc[u] = vc[u] = 0;
                _Pragma("unroll") for (int j = 0; j < kVec; ++j) {
                    const uint32_t r = mix(x + j * 0x9E3779B1u);
                    /* a root that is not 0 keeps the smallest code: 2^-9 and any dither give it */
                    const float y = root[j] > 0.0f ? fmaxf(root[j] * sv, 0x1p-9f) : 0.0f;
                    mc[u] = put_code(m[u][j] * sm, r & 0xffff0000u, mc[u], j);
                    vc[u] = put_code(y, r << 16, vc[u], j);
                }
                if (me[u] == 255u) mc[u] = 0x7f7f7f7fu; /* a block with an infinity or NaN is NaN */
                if (ve[u] == 255u) vc[u] = 0x7f7f7f7fu;
                if (!kWhole) { /* codes behind the tensor's end stay zeros */
                    const uint32_t keep = left >= 4 ? ~0u : left > 0 ? (1u << (8 * left)) - 1u : 0u;
                    mc[u] &= keep, vc[u] &= keep;
                }
                if (kWhole || left > 0) {
                    *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.m) + k) = mc[u];
                    *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.v) + k) = vc[u];
                    if (k % kGroup == 0) a.m_exp[k / kGroup] = (uint8_t)me[u], a.v_exp[k / kGroup] = (uint8_t)ve[u];
                }
            } else {
                store_quad<float, kWhole, kStream>(static_cast<float*>(a.m) + k, left, m[u]);
                store_quad<float, kWhole, kStream>(static_cast<float*>(a.v) + k, left, v[u]);
            }
            store_quad<P, kWhole, kStream>(param + i, left, w[u]);
            if (master) store_quad<float, kWhole, kStream>(a.master + k, left, w[u]);
        }
    }
}

/* kStream: everything but the byte codes past the caches.  For lists whose arrays do not fit the 256 MiB last-level cache together, where
 * what a step leaves there only pushes out what it still has to read: 100M bf16 + fp32 master 500 -> 452 us (and the norm in front of
 * it 71 -> 37); 16M fp32, which fits, 70 us without and 80 with. */
template <typename P, typename G, bool kBytes, bool kStream>
__global__ void __launch_bounds__(kBlock) k_adamw(const StepArgs a) {
    const Control c = *a.control;
    if (c.skip) return;
    for (int64_t tile = blockIdx.x; tile < a.n_tiles; tile += gridDim.x) {
        const int which = find_tensor(a.params, a.n, tile);
        const Entry e = a.params[which];
        const G* grad = static_cast<const G*>(a.grads[which].data);
        if (!e.data || !grad) continue;
        const int64_t from = (tile - e.first_tile) * kTile;
        P* param = static_cast<P*>(e.data) + from;
        if (e.count - from >= kTile) step_tile<P, G, kBytes, true, kBlock, kStream>(a, c, param, grad + from, e.state_at + from, kTile);
        else step_tile<P, G, kBytes, false, kBlock, kStream>(a, c, param, grad + from, e.state_at + from, (int)(e.count - from));
    }
}

/* The whole step of a short list in one launch: block b updates tile b, and every block takes the norm of all of them by itself (a
 * wave a tile), for it has less to read than another launch costs: a clipped step of the CartPole MLP's 16 tensors 9.3 us, 15.5 by three
 * launches.  As many tiles as a block of 1024 threads has waves: fp32 tensors of 4096, one 6.2 us here and 10.0 there, 8 of them 7.3 and 10.6,
 * 16 8.0 and 11.3 (in a graph 7.9 and 9.0); with a 17th three launches take 12.1 (9.1).
 * The step counter moves when every block has read it. */
template <typename P, typename G, bool kBytes>
__global__ void __launch_bounds__(kSmallBlock) k_adamw_small(const StepArgs a, int norm_here) {
    __shared__ double lds[kSmallTiles];
    __shared__ Control shared;
    const int wave = threadIdx.x >> 6;
    if (norm_here) {
        double sum = 0.0;
        if (wave < a.n_tiles) {
            const Entry e = a.grads[find_tensor(a.grads, a.n, wave)];
            const int64_t from = (wave - e.first_tile) * kTile, to = from + kTile;
            if (e.data) sum = sum_squares<G, false>(static_cast<const G*>(e.data), from, to < e.count ? to : e.count, threadIdx.x & 63, 64);
        }
        for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
        if ((threadIdx.x & 63) == 0) lds[wave] = sum;
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        float norm = 0.0f;
        if (norm_here) {
            double sum = 0.0;
            for (int w = 0; w < kSmallTiles; ++w) sum += lds[w];
            norm = (float)(fabs(a.grad_scale) * sqrt(sum));
        } else if (a.max_norm > 0.0) {
            norm = a.norm[0];
        }
        const int t = a.control->step + 1;
        Control c;
        const bool go = step_values(a, norm, t, c);
        shared = c;
        if (__hip_atomic_fetch_add(&a.control->ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1) {
            if (go) a.control->step = t;
            else a.control->skipped += 1;
            if (norm_here && a.norm) a.norm[0] = norm;
            a.control->skip = c.skip;
            a.control->ticket = 0;
        }
    }
    __syncthreads();
    const Control c = shared;
    if (c.skip) return;
    const int which = find_tensor(a.params, a.n, blockIdx.x);
    const Entry e = a.params[which];
    const G* grad = static_cast<const G*>(a.grads[which].data);
    if (!e.data || !grad) return;
    const int64_t from = (blockIdx.x - e.first_tile) * kTile;
    P* param = static_cast<P*>(e.data) + from;
    if (e.count - from >= kTile) step_tile<P, G, kBytes, true, kSmallBlock, false>(a, c, param, grad + from, e.state_at + from, kTile);
    else step_tile<P, G, kBytes, false, kSmallBlock, false>(a, c, param, grad + from, e.state_at + from, (int)(e.count - from));
}

int norm_blocks(int64_t n_tiles) { return (int)(n_tiles < kMaxPartials ? n_tiles : kMaxPartials); }

template <typename G>
void launch_norm(const Entry* table, int n, int64_t n_tiles, bool stream, double* partial, hipStream_t st) {
    const dim3 grid((unsigned)norm_blocks(n_tiles)), block(kBlock);
    if (stream) hipLaunchKernelGGL((k_norm_partial<G, true>), grid, block, 0, st, table, n, n_tiles, partial);
    else hipLaunchKernelGGL((k_norm_partial<G, false>), grid, block, 0, st, table, n, n_tiles, partial);
}
constexpr double kCache = 256.0 * 1048576.0; /* bytes of the last-level cache */
void launch_norm(const Entry* table, int n, int64_t n_tiles, int dtype, bool alone, double* partial, hipStream_t st) {
    const bool stream = alone && (double)n_tiles * kTile * (dtype == MZS_DTYPE_FLOAT ? 4 : 2) > kCache;
    if (dtype == MZS_DTYPE_FLOAT) launch_norm<float>(table, n, n_tiles, stream, partial, st);
    else if (dtype == MZS_DTYPE_BFLOAT) launch_norm<bf16>(table, n, n_tiles, stream, partial, st);
    else launch_norm<_Float16>(table, n, n_tiles, stream, partial, st);
}

struct Launch {
    StepArgs s;
    int bits, norm_here; /* -1: the two-launch way */
    hipStream_t st;
};
template <typename P, typename G>
void launch_step(const Launch& l) {
    if (l.norm_here >= 0) {
        const dim3 grid((unsigned)l.s.n_tiles), block(kSmallBlock);
        if (l.bits == 8) hipLaunchKernelGGL((k_adamw_small<P, G, true>), grid, block, 0, l.st, l.s, l.norm_here);
        else hipLaunchKernelGGL((k_adamw_small<P, G, false>), grid, block, 0, l.st, l.s, l.norm_here);
        return;
    }
    const dim3 grid((unsigned)(l.s.n_tiles < 65536 ? l.s.n_tiles : 65536)), block(kBlock);
    const double each = sizeof(P) + sizeof(G) + (l.s.master ? 4 : 0) + (l.bits == 8 ? 2.0625 : 8.0);
    const bool stream = each * kTile * (double)l.s.n_tiles > kCache;
    if (l.bits == 8 && stream) hipLaunchKernelGGL((k_adamw<P, G, true, true>), grid, block, 0, l.st, l.s);
    else if (l.bits == 8) hipLaunchKernelGGL((k_adamw<P, G, true, false>), grid, block, 0, l.st, l.s);
    else if (stream) hipLaunchKernelGGL((k_adamw<P, G, false, true>), grid, block, 0, l.st, l.s);
    else hipLaunchKernelGGL((k_adamw<P, G, false, false>), grid, block, 0, l.st, l.s);
}
template <typename P>
void launch_step(const Launch& l, int grad_dtype) {
    if (grad_dtype == MZS_DTYPE_FLOAT) launch_step<P, float>(l);
    else if (grad_dtype == MZS_DTYPE_BFLOAT) launch_step<P, bf16>(l);
    else launch_step<P, _Float16>(l);
}

bool known_dtype(int t) { return t >= MZS_DTYPE_FLOAT && t <= MZS_DTYPE_HALF; }

}  // namespace
}  // namespace mzs

using namespace mzs;

extern "C" {

int mzs_optim_table(int32_t device, int32_t n, const void* const* pointers, const int64_t* counts, void* table_dev,
                    int64_t* n_tiles_out, void* stream) {
    if (n < 0 || !table_dev || !n_tiles_out || (n > 0 && (!pointers || !counts))) return set_error(MZS_E_ARG, "null argument");
    for (int32_t i = 0; i < n; ++i)
        if (counts[i] < 0 || counts[i] > ((int64_t)1 << 48)) return set_error(MZS_E_ARG, "tensor size");
    DeviceScope scope(device);
    if (scope.status != hipSuccess) return hip_error("mzs_optim_table: device", scope.status);
    int64_t tile = 0, at = 0;
    for (int32_t from = 0; from <= n; from += kFillEntries) { /* entry n closes the table */
        FillArgs a;
        const int m = n + 1 - from < kFillEntries ? n + 1 - from : kFillEntries;
        for (int j = 0; j < m; ++j) {
            const int32_t i = from + j;
            Entry& e = a.entries[j];
            e.data = i < n && counts[i] ? const_cast<void*>(pointers[i]) : nullptr;
            e.count = i < n ? counts[i] : 0;
            e.first_tile = tile;
            e.state_at = at;
            tile += (e.count + kTile - 1) / kTile;
            at += (e.count + MZS_OPTIM_ALIGN - 1) / MZS_OPTIM_ALIGN * MZS_OPTIM_ALIGN;
        }
        hipLaunchKernelGGL(k_optim_table, dim3(1), dim3(128), 0, static_cast<hipStream_t>(stream), a,
                           static_cast<Entry*>(table_dev), from, m);
    }
    *n_tiles_out = tile;
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MZS_OK : hip_error("mzs_optim_table: launch", e);
}

size_t mzs_grad_norm_workspace(int64_t n_tiles) { return sizeof(double) * (size_t)(n_tiles > 0 ? norm_blocks(n_tiles) : 1); }

int mzs_grad_norm(int32_t device, int32_t n, const void* table_dev, int64_t n_tiles, int32_t dtype, double grad_scale,
                  float* norm_dev, void* workspace, size_t workspace_bytes, void* stream) {
    if (n < 0 || n_tiles < 0 || !table_dev || !norm_dev || !workspace) return set_error(MZS_E_ARG, "null argument");
    if (!known_dtype(dtype)) return set_error(MZS_E_ARG, "gradients: fp32, bf16 or fp16");
    if (!(std::fabs(grad_scale) < HUGE_VAL)) return set_error(MZS_E_ARG, "grad_scale must be finite");
    if (workspace_bytes < mzs_grad_norm_workspace(n_tiles)) return set_error(MZS_E_ARG, "workspace too small (mzs_grad_norm_workspace)");
    DeviceScope scope(device);
    if (scope.status != hipSuccess) return hip_error("mzs_grad_norm: device", scope.status);
    hipStream_t st = static_cast<hipStream_t>(stream);
    double* partial = static_cast<double*>(workspace);
    if (n_tiles > 0) launch_norm(static_cast<const Entry*>(table_dev), n, n_tiles, dtype, true, partial, st);
    hipLaunchKernelGGL(k_norm_join, dim3(1), dim3(kBlock), 0, st, (const double*)partial, n_tiles > 0 ? norm_blocks(n_tiles) : 0,
                       std::fabs(grad_scale), norm_dev);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MZS_OK : hip_error("mzs_grad_norm: launch", e);
}

int mzs_adamw_step(const mzs_adamw_args* a, void* stream) {
    if (!a || a->n < 0 || a->n_tiles < 0 || !a->params_table || !a->grads_table || !a->control_dev)
        return set_error(MZS_E_ARG, "null argument");
    if (!known_dtype(a->param_dtype) || !known_dtype(a->grad_dtype)) return set_error(MZS_E_ARG, "parameters and gradients: fp32, bf16 or fp16");
    if (a->state_bits != 32 && a->state_bits != 8) return set_error(MZS_E_ARG, "state_bits: 32 or 8");
    if (a->n_tiles > 0 && (!a->exp_avg || !a->exp_avg_sq || (a->state_bits == 8 && (!a->exp_avg_exponent || !a->exp_avg_sq_exponent))))
        return set_error(MZS_E_ARG, "null state");
    if (!(a->beta1 >= 0.0 && a->beta1 < 1.0 && a->beta2 >= 0.0 && a->beta2 < 1.0)) return set_error(MZS_E_ARG, "betas must be in [0, 1)");
    if (!(a->eps >= 0.0) || !(a->weight_decay >= 0.0) || !(a->max_norm >= 0.0) || !(std::fabs(a->grad_scale) < HUGE_VAL) ||
        (!a->lr_dev && !(a->lr >= 0.0)))
        return set_error(MZS_E_ARG, "lr, eps, weight_decay, max_norm >= 0 and a finite grad_scale");
    const bool compute = a->max_norm > 0.0 && !a->norm_given;
    if (a->max_norm > 0.0 && a->norm_given && !a->norm_dev) return set_error(MZS_E_ARG, "norm_given without norm_dev");
    if (compute && (!a->workspace || a->workspace_bytes < mzs_grad_norm_workspace(a->n_tiles)))
        return set_error(MZS_E_ARG, "workspace too small (mzs_grad_norm_workspace)");
    DeviceScope scope(a->device);
    if (scope.status != hipSuccess) return hip_error("mzs_adamw_step: device", scope.status);
    hipStream_t st = static_cast<hipStream_t>(stream);
    StepArgs s;
    s.params = static_cast<const Entry*>(a->params_table), s.grads = static_cast<const Entry*>(a->grads_table);
    s.master = a->master, s.m = a->exp_avg, s.v = a->exp_avg_sq, s.m_exp = a->exp_avg_exponent, s.v_exp = a->exp_avg_sq_exponent;
    s.control = reinterpret_cast<Control*>(a->control_dev);
    s.norm = a->norm_dev, s.lr_dev = a->lr_dev;
    s.partial = static_cast<const double*>(a->workspace);
    s.n_tiles = a->n_tiles;
    s.lr = a->lr, s.beta1 = a->beta1, s.beta2 = a->beta2, s.weight_decay = a->weight_decay, s.max_norm = a->max_norm;
    s.grad_scale = a->grad_scale, s.seed = a->seed;
    s.b1 = (float)a->beta1, s.one_minus_b1 = (float)(1.0 - a->beta1);
    s.b2 = (float)a->beta2, s.one_minus_b2 = (float)(1.0 - a->beta2);
    s.eps = (float)a->eps;
    s.n = a->n;
    s.n_partial = 0;
    if (compute && a->n_tiles == 0) return set_error(MZS_E_ARG, "no tensors to take a norm of");
    const bool small = a->n_tiles > 0 && a->n_tiles <= kSmallTiles;
    if (!small) {
        if (compute) {
            s.n_partial = norm_blocks(a->n_tiles);
            launch_norm(s.grads, a->n, a->n_tiles, a->grad_dtype, false, static_cast<double*>(a->workspace), st);
        }
        hipLaunchKernelGGL(k_adamw_begin, dim3(1), dim3(kBlock), 0, st, s);
    }
    if (a->n_tiles > 0) {
        const Launch l{s, a->state_bits, small ? (int)compute : -1, st};
        if (a->param_dtype == MZS_DTYPE_FLOAT) launch_step<float>(l, a->grad_dtype);
        else if (a->param_dtype == MZS_DTYPE_BFLOAT) launch_step<bf16>(l, a->grad_dtype);
        else launch_step<_Float16>(l, a->grad_dtype);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MZS_OK : hip_error("mzs_adamw_step: launch", e);
}

}  // extern "C"
