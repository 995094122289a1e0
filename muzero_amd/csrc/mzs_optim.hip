/*
 * mzs_optim.hip — global gradient norm and AdamW step over many tensors (include/mzsearch.h, mzs_optim_*, mzs_grad_norm,
 * mzs_adamw_step).
 *
 * Work is cut into tiles of kTile elements of one tensor; a table in device memory says which tensor a tile is of.
 */
#include "mzs_error.h"

#include <cmath>
#include <cstdint>
#include <cstring>

namespace mzs {
namespace {

constexpr int kBlock = 256;
constexpr int kTile = 4096;       /* elements of a tile */
constexpr int kFillEntries = 120; /* table entries a launch carries in its arguments */
constexpr int kMaxPartials = 1024;
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
__device__ __forceinline__ void put(bf16* p, float v) { /* nearest even; a NaN stays one */
    uint32_t b = __float_as_uint(v);
    b = v != v ? 0x7fc00000u : b + 0x7fffu + ((b >> 16) & 1u);
    p->bits = (uint16_t)(b >> 16);
}
__device__ __forceinline__ void put(_Float16* p, float v) { *p = (_Float16)v; }

/* the tensor that tile `tile` is of: the last entry with first_tile <= tile (empty tensors have no tiles) */
__device__ __forceinline__ int find_tensor(const Entry* __restrict__ table, int n, int64_t tile) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (table[mid].first_tile <= tile) lo = mid;
        else hi = mid;
    }
    return lo;
}

/* fixed-order sum over the block; the total in thread 0 */
__device__ __forceinline__ double block_sum(double v, double* lds) {
    lds[threadIdx.x] = v;
    __syncthreads();
    for (int w = kBlock / 2; w > 0; w >>= 1) {
        if ((int)threadIdx.x < w) lds[threadIdx.x] += lds[threadIdx.x + w];
        __syncthreads();
    }
    return lds[0];
}

template <typename G>
__global__ void __launch_bounds__(kBlock) k_norm_partial(const Entry* __restrict__ table, int n, int64_t n_tiles,
                                                         double* __restrict__ partial) {
    __shared__ double lds[kBlock];
    double sum = 0.0;
    for (int64_t tile = blockIdx.x; tile < n_tiles; tile += gridDim.x) {
        const Entry e = table[find_tensor(table, n, tile)];
        if (!e.data) continue;
        const int64_t from = (tile - e.first_tile) * kTile;
        const int64_t to = from + kTile < e.count ? from + kTile : e.count;
        const G* g = static_cast<const G*>(e.data);
        for (int64_t i = from + threadIdx.x; i < to; i += kBlock) {
            const double x = (double)to_float(g[i]);
            sum = fma(x, x, sum);
        }
    }
    const double total = block_sum(sum, lds);
    if (threadIdx.x == 0) partial[blockIdx.x] = total;
}

struct Control {
    int32_t step, skipped;
    int32_t skip;       /* this step is skipped               */
    uint32_t key;       /* dither key of this step            */
    float scale;        /* grad_scale * clip                  */
    float step_size;    /* lr / (1 - beta1^t)                 */
    float decay;        /* 1 - lr * weight_decay              */
    float inv_root_2;   /* 1 / sqrt(1 - beta2^t)              */
};
static_assert(sizeof(Control) <= MZS_OPTIM_CONTROL_BYTES, "control size");

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
    __shared__ double lds[kBlock];
    const double total = join_partials(partial, n, lds);
    if (threadIdx.x == 0) norm[0] = (float)(scale * sqrt(total));
}

/* one block before the update: the norm (joined from n_partial sums, or given), clipping, bias corrections, the step counter */
__global__ void __launch_bounds__(kBlock) k_adamw_begin(const StepArgs a) {
    __shared__ double lds[kBlock];
    float norm = 0.0f;
    if (a.n_partial > 0) {
        norm = (float)(fabs(a.grad_scale) * sqrt(join_partials(a.partial, a.n_partial, lds)));
        if (threadIdx.x == 0 && a.norm) a.norm[0] = norm;
    } else if (a.max_norm > 0.0) {
        norm = a.norm[0];
    }
    if (threadIdx.x != 0) return;
    Control* c = a.control;
    const bool skip = a.max_norm > 0.0 && !(fabsf(norm) < __builtin_inff());
    c->skip = skip;
    if (skip) {
        c->skipped += 1;
        return;
    }
    const int t = c->step + 1;
    const double lr = a.lr_dev ? (double)a.lr_dev[0] : a.lr;
    float clip = 1.0f;
    if (a.max_norm > 0.0) clip = fminf(1.0f, (float)a.max_norm / (norm + 1e-6f));
    c->step = t;
    c->key = mix((uint32_t)a.seed ^ mix((uint32_t)t * 0x9E3779B9u + (uint32_t)(a.seed >> 32)));
    c->scale = (float)a.grad_scale * clip;
    c->step_size = (float)(lr / (1.0 - pow(a.beta1, (double)t)));
    c->decay = (float)(1.0 - lr * a.weight_decay);
    c->inv_root_2 = (float)(1.0 / sqrt(1.0 - pow(a.beta2, (double)t)));
}

/* ---- 8-bit states: e4m3 codes under a shared power of two */
__device__ __forceinline__ float code_value(uint8_t code) {
    const uint32_t mag = code & 0x7fu, e = mag >> 3, f = mag & 7u;
    float v = e ? __uint_as_float(((e + 120u) << 23) | (f << 20)) : (float)f * 0.001953125f;
    if (mag == 0x7fu) v = __builtin_nanf("");
    return (code & 0x80u) ? -v : v;
}
__device__ __forceinline__ float exponent_value(uint8_t e) { /* 2^(e - 127); 255: NaN */
    return e == 255 ? __builtin_nanf("") : e ? __uint_as_float((uint32_t)e << 23) : 5.87747175411143754e-39f;
}
/* exponent byte of a block whose largest magnitude is `most` */
__device__ __forceinline__ uint8_t block_exponent(float most) {
    const uint32_t b = __float_as_uint(most);
    if (b >= 0x7f800000u) return 255;
    const int e = (int)((b + 0x1fffffu) >> 23) - 8; /* 448 = 1.75 * 2^8: a mantissa above 1.75 carries */
    return (uint8_t)(e < 0 ? 0 : e);
}
/* |y| <= 448 to a code: the grid point below |y| / step + r steps, r in [0, 1) */
__device__ __forceinline__ uint8_t to_code(float y, float r) {
    if (y != y) return 0x7f;
    const float a = fabsf(y);
    const int e = (int)(__float_as_uint(a) >> 23) - 127;
    const int oct = e < -6 ? -6 : e;
    const float inv_step = __uint_as_float((uint32_t)(127 - (oct - 3)) << 23);
    int q = (int)floorf(a * inv_step + r); /* 8 .. 16 in a normal octave, 0 .. 8 below */
    uint32_t code = oct == -6 ? (uint32_t)q : (uint32_t)(((oct + 6) << 3) + q);
    return (uint8_t)(code | ((__float_as_uint(y) >> 24) & 0x80u));
}

__device__ __forceinline__ float adamw(float w, float& m, float& v, float& root, float g, const StepArgs& a, const Control& c) {
    m = m * a.b1 + g * a.one_minus_b1;
    v = v * a.b2 + g * g * a.one_minus_b2;
    root = __builtin_sqrtf(v);
    return w * c.decay - c.step_size * (m / (root * c.inv_root_2 + a.eps));
}

template <typename P, typename G, bool kBytes>
__global__ void __launch_bounds__(kBlock) k_adamw(const StepArgs a) {
    const Control c = *a.control;
    if (c.skip) return;
    for (int64_t tile = blockIdx.x; tile < a.n_tiles; tile += gridDim.x) {
        const int which = find_tensor(a.params, a.n, tile);
        const Entry e = a.params[which];
        const G* grad = static_cast<const G*>(a.grads[which].data);
        if (!e.data || !grad) continue;
        const int64_t from = (tile - e.first_tile) * kTile;
        const int64_t to = from + kTile < e.count ? from + kTile : e.count;
        P* param = static_cast<P*>(e.data);
        for (int64_t i0 = from; i0 < to; i0 += kBlock) {
            const int64_t i = i0 + threadIdx.x, k = e.state_at + i;
            const bool live = i < to;
            float m = 0.0f, v = 0.0f, root = 0.0f;
            uint8_t mb = 0, vb = 0;
            if (kBytes) { /* the 32 lanes of a block share their exponents; those behind the tensor's end count as zero */
                if (live) {
                    mb = a.m_exp[k / kGroup], vb = a.v_exp[k / kGroup];
                    m = code_value(static_cast<const uint8_t*>(a.m)[k]) * exponent_value(mb);
                    const float u = code_value(static_cast<const uint8_t*>(a.v)[k]) * exponent_value(vb);
                    v = u * u;
                }
            } else if (live) {
                m = static_cast<const float*>(a.m)[k], v = static_cast<const float*>(a.v)[k];
            }
            if (live) {
                const float g = to_float(grad[i]) * c.scale;
                const float w = adamw(a.master ? a.master[k] : to_float(param[i]), m, v, root, g, a, c);
                put(param + i, w);
                if (a.master) a.master[k] = w;
            }
            if (kBytes) {
                float most_m = fabsf(m), most_u = root;
                for (int off = 16; off > 0; off >>= 1) { /* NaN wins: compared as bits */
                    const uint32_t om = __float_as_uint(__shfl_xor(most_m, off, 64)), ou = __float_as_uint(__shfl_xor(most_u, off, 64));
                    most_m = __uint_as_float(max(__float_as_uint(most_m), om));
                    most_u = __uint_as_float(max(__float_as_uint(most_u), ou));
                }
                mb = block_exponent(most_m), vb = block_exponent(most_u);
                if (live) {
                    const uint32_t r = mix((uint32_t)k * 0x9E3779B1u + c.key);
                    const float rm = (float)(r >> 16) * 0x1p-16f, rv = (float)(r & 0xffffu) * 0x1p-16f;
                    const float sm = __uint_as_float((254u - mb) << 23), sv = __uint_as_float((254u - vb) << 23);
                    const uint8_t cm = mb == 255 ? 0x7f : to_code(m * sm, rm);
                    uint8_t cv = vb == 255 ? 0x7f : to_code(root * sv, rv);
                    if (cv == 0 && root > 0.0f) cv = 1;
                    static_cast<uint8_t*>(a.m)[k] = cm;
                    static_cast<uint8_t*>(a.v)[k] = cv;
                    if (k % kGroup == 0) a.m_exp[k / kGroup] = mb, a.v_exp[k / kGroup] = vb;
                }
            } else if (live) {
                static_cast<float*>(a.m)[k] = m, static_cast<float*>(a.v)[k] = v;
            }
        }
    }
}

int norm_blocks(int64_t n_tiles) { return (int)(n_tiles < kMaxPartials ? n_tiles : kMaxPartials); }

void launch_norm(const Entry* table, int n, int64_t n_tiles, int dtype, double* partial, hipStream_t st) {
    const dim3 grid((unsigned)norm_blocks(n_tiles)), block(kBlock);
    if (dtype == MZS_DTYPE_FLOAT) hipLaunchKernelGGL(k_norm_partial<float>, grid, block, 0, st, table, n, n_tiles, partial);
    else if (dtype == MZS_DTYPE_BFLOAT) hipLaunchKernelGGL(k_norm_partial<bf16>, grid, block, 0, st, table, n, n_tiles, partial);
    else hipLaunchKernelGGL(k_norm_partial<_Float16>, grid, block, 0, st, table, n, n_tiles, partial);
}

template <typename P, typename G>
void launch_step(const StepArgs& s, int bits, hipStream_t st) {
    const dim3 grid((unsigned)(s.n_tiles < 65536 ? s.n_tiles : 65536)), block(kBlock);
    if (bits == 8) hipLaunchKernelGGL((k_adamw<P, G, true>), grid, block, 0, st, s);
    else hipLaunchKernelGGL((k_adamw<P, G, false>), grid, block, 0, st, s);
}
template <typename P>
void launch_step(const StepArgs& s, int grad_dtype, int bits, hipStream_t st) {
    if (grad_dtype == MZS_DTYPE_FLOAT) launch_step<P, float>(s, bits, st);
    else if (grad_dtype == MZS_DTYPE_BFLOAT) launch_step<P, bf16>(s, bits, st);
    else launch_step<P, _Float16>(s, bits, st);
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
    if (n_tiles > 0) launch_norm(static_cast<const Entry*>(table_dev), n, n_tiles, dtype, partial, st);
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
    if (compute && a->n_tiles > 0) {
        s.n_partial = norm_blocks(a->n_tiles);
        launch_norm(s.grads, a->n, a->n_tiles, a->grad_dtype, static_cast<double*>(a->workspace), st);
    } else if (compute) {
        return set_error(MZS_E_ARG, "no tensors to take a norm of");
    }
    hipLaunchKernelGGL(k_adamw_begin, dim3(1), dim3(kBlock), 0, st, s);
    if (a->n_tiles > 0) {
        if (a->param_dtype == MZS_DTYPE_FLOAT) launch_step<float>(s, a->grad_dtype, a->state_bits, st);
        else if (a->param_dtype == MZS_DTYPE_BFLOAT) launch_step<bf16>(s, a->grad_dtype, a->state_bits, st);
        else launch_step<_Float16>(s, a->grad_dtype, a->state_bits, st);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MZS_OK : hip_error("mzs_adamw_step: launch", e);
}

}  // extern "C"
