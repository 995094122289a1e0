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

#include <cstdint>

namespace mzs {
namespace {

constexpr float kLn2 = 0.69314718055994530942f;
constexpr double kLog2e = 1.44269504088896340736;
constexpr float kLow = -1e30f; /* stands for -inf where it is multiplied by an exponential that is 0 */

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
    float scale; /* inverse_temperature              */
    float c;     /* inverse_temperature * log2 e     */
};

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) {
    return v;
}
struct bf16 {
    uint16_t bits;
};
template <>
__device__ __forceinline__ float to_float<bf16>(bf16 v) {
    return __uint_as_float((uint32_t)v.bits << 16);
}
template <>
__device__ __forceinline__ float to_float<_Float16>(_Float16 v) {
    return (float)v;
}
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ bf16 from_float<bf16>(float v) { /* round to nearest even; a NaN stays one */
    uint32_t b = __float_as_uint(v);
    b = v != v ? 0x7fc00000u : b + 0x7fffu + ((b >> 16) & 1u);
    return bf16{(uint16_t)(b >> 16)};
}
template <>
__device__ __forceinline__ _Float16 from_float<_Float16>(float v) {
    return (_Float16)v;
}

/* one part of a row: its largest logit, and s and t relative to it */
struct Sum {
    float big, s, t;
};

__device__ __forceinline__ Sum sum_merge(Sum a, Sum b, float c) {
    const float big = fmaxf(a.big, b.big);
    const float da = a.big == big ? 0.0f : fmaxf(c * (a.big - big), kLow);
    const float db = b.big == big ? 0.0f : fmaxf(c * (b.big - big), kLow);
    const float fa = __builtin_amdgcn_exp2f(da), fb = __builtin_amdgcn_exp2f(db);
    return Sum{big, fa * a.s + fb * b.s, fa * (a.t + da * a.s) + fb * (b.t + db * b.s)};
}

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

constexpr int kBlock = 256;

__device__ __forceinline__ void write_row(const Row& p, int64_t r, Sum v, float l_action, int64_t a) {
    const bool empty = v.s == 0.0f;
    const float log2_s = log2f(v.s), log_total = kLn2 * log2_s;
    p.log_z[r] = empty ? -__builtin_inff() : p.scale * v.big + log_total;
    p.entropy[r] = empty ? 0.0f : kLn2 * (log2_s - v.t / v.s);
    p.row_stats[2 * r] = v.big;
    p.row_stats[2 * r + 1] = v.s;
    float lp = 0.0f;
    if (a >= p.n) lp = __builtin_nanf("");
    else if (a >= 0) lp = empty ? -__builtin_inff() : p.scale * (l_action - v.big) - log_total;
    p.log_prob[r] = lp;
}

/* One block per row, one logit a thread and step. */
template <typename T>
__global__ void __launch_bounds__(kBlock) k_policy_rows(const Row p) {
    __shared__ Sum parts[kBlock];
    __shared__ uint64_t keys[kBlock];
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T* l = static_cast<const T*>(p.logits) + r * p.logits_stride;
        const uint8_t* mask = p.mask ? p.mask + r * p.mask_stride : nullptr;
        Sum v{-__builtin_inff(), 0.0f, 0.0f};
        for (int64_t i = threadIdx.x; i < p.n; i += kBlock) {
            if (mask && !mask[i]) continue;
            const float x = to_float(l[i]);
            if (x == -__builtin_inff()) continue;
            v = sum_merge(v, Sum{x != x ? v.big : x, x != x ? x : 1.0f, 0.0f}, p.c);
        }
        parts[threadIdx.x] = v;
        __syncthreads();
        for (int w = kBlock / 2; w > 0; w >>= 1) {
            if (threadIdx.x < (unsigned)w) parts[threadIdx.x] = sum_merge(parts[threadIdx.x], parts[threadIdx.x + w], p.c);
            __syncthreads();
        }
        v = parts[0];
        if (v.big == __builtin_inff()) v.s = __builtin_nanf("");
        if (threadIdx.x == 0) {
            const int64_t a = row_action(p, r);
            const float la = a < 0 || a >= p.n ? 0.0f : mask && !mask[a] ? -__builtin_inff() : to_float(l[a]);
            write_row(p, r, v, la, a);
        }
        uint64_t last = ~0ull;
        for (int k = 0; k < p.top; ++k) {
            uint64_t best = 0;
            for (int64_t i = threadIdx.x; i < p.n; i += kBlock) {
                if (mask && !mask[i]) continue;
                const float x = to_float(l[i]);
                const uint64_t key = x == -__builtin_inff() ? 0 : rank_key(x, (uint32_t)i);
                if (key < last && key > best) best = key;
            }
            keys[threadIdx.x] = best;
            __syncthreads();
            for (int w = kBlock / 2; w > 0; w >>= 1) {
                if (threadIdx.x < (unsigned)w && keys[threadIdx.x + w] > keys[threadIdx.x])
                    keys[threadIdx.x] = keys[threadIdx.x + w];
                __syncthreads();
            }
            last = keys[0];
            if (threadIdx.x == 0) {
                const float log_total = kLn2 * log2f(v.s);
                p.top_action[r * p.top + k] = last ? (int32_t)(0xffffffffu - (uint32_t)last) : -1;
                p.top_log_prob[r * p.top + k] =
                    last ? p.scale * (key_value(last) - v.big) - log_total : -__builtin_inff();
            }
            __syncthreads();
        }
        __syncthreads();
    }
}

template <typename T>
__global__ void __launch_bounds__(kBlock) k_policy_grad(const Row p) {
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T* l = static_cast<const T*>(p.logits) + r * p.logits_stride;
        const uint8_t* mask = p.mask ? p.mask + r * p.mask_stride : nullptr;
        T* g = static_cast<T*>(p.grad_logits) + r * p.grad_stride;
        const int64_t a = row_action(p, r);
        const float big = p.row_stats[2 * r], s = p.row_stats[2 * r + 1];
        const bool empty = s == 0.0f;
        const float log2_s = log2f(s);
        const float ga = a < 0 || !p.grad_log_prob ? 0.0f : a >= p.n ? __builtin_nanf("") : p.grad_log_prob[r];
        const float gh = p.grad_entropy ? p.grad_entropy[r] : 0.0f, gz = p.grad_log_z ? p.grad_log_z[r] : 0.0f;
        const float base = gz - ga - gh * p.entropy[r];
        for (int64_t i = threadIdx.x; i < p.n; i += kBlock) {
            const float x = to_float(l[i]);
            float out = 0.0f;
            if (!empty && !(mask && !mask[i]) && x != -__builtin_inff()) {
                const float d = fmaxf(p.c * (x - big), kLow), e = x != x ? x : __builtin_amdgcn_exp2f(d);
                out = e / s * (base - gh * (kLn2 * (d - log2_s)));
                if (i == a) out += ga;
                out *= p.scale;
            }
            g[i] = from_float<T>(out);
        }
    }
}

int check(const mzs_policy_args* a, bool forward, bool grad) {
    if (!a) return set_error(MZS_E_ARG, "null arguments");
    if (a->dtype < MZS_DTYPE_FLOAT || a->dtype > MZS_DTYPE_HALF) return set_error(MZS_E_ARG, "logits: fp32, bf16 or fp16");
    if (a->rows < 0 || a->n_actions < 1 || a->n_actions > 0x7fffffff) return set_error(MZS_E_ARG, "rows >= 0 and 1 <= n_actions < 2^31");
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
    p.scale = a.inverse_temperature;
    p.c = (float)((double)a.inverse_temperature * kLog2e);
    return p;
}

unsigned row_grid(int64_t rows) { return (unsigned)(rows < 65536 ? rows : 65536); }

template <typename T>
void launch_rows(const Row& p, hipStream_t st) {
    hipLaunchKernelGGL(k_policy_rows<T>, dim3(row_grid(p.rows)), dim3(kBlock), 0, st, p);
}
template <typename T>
void launch_grad(const Row& p, hipStream_t st) {
    hipLaunchKernelGGL(k_policy_grad<T>, dim3(row_grid(p.rows)), dim3(kBlock), 0, st, p);
}

int run(const mzs_policy_args* a, void* stream, bool forward, bool grad) {
    const int rc = check(a, forward, grad);
    if (rc || a->rows == 0) return rc;
    DeviceScope scope(a->device);
    if (scope.status != hipSuccess) return hip_error("mzs_policy: device", scope.status);
    const Row p = pack(*a);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (forward) {
        if (a->dtype == MZS_DTYPE_FLOAT) launch_rows<float>(p, st);
        else if (a->dtype == MZS_DTYPE_BFLOAT) launch_rows<bf16>(p, st);
        else launch_rows<_Float16>(p, st);
    }
    if (grad) {
        if (a->dtype == MZS_DTYPE_FLOAT) launch_grad<float>(p, st);
        else if (a->dtype == MZS_DTYPE_BFLOAT) launch_grad<bf16>(p, st);
        else launch_grad<_Float16>(p, st);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MZS_OK : hip_error("mzs_policy: launch", e);
}

}  // namespace
}  // namespace mzs

extern "C" {

int mzs_policy_workspace(const mzs_policy_args* args, size_t* bytes_out) {
    if (!args || !bytes_out) return mzs::set_error(MZS_E_ARG, "null argument");
    *bytes_out = 0;
    return MZS_OK;
}
int mzs_policy_log_probs(const mzs_policy_args* args, void* stream) { return mzs::run(args, stream, true, false); }
int mzs_policy_log_probs_grad(const mzs_policy_args* args, void* stream) { return mzs::run(args, stream, false, true); }
int mzs_policy_log_probs_train(const mzs_policy_args* args, void* stream) { return mzs::run(args, stream, true, true); }

}  // extern "C"
