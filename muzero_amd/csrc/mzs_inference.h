/*
 * mzs_inference.h — the standalone inference kernel (k_inference) and a wave's LDS slice, for the units that instantiate it:
 * mzsearch.hip, and mzs_logits.hip for the form that writes the policy head's logits.
 */
#ifndef MZS_INFERENCE_H
#define MZS_INFERENCE_H

#include "mzs_search_kernels.h"

namespace mzs {

__device__ __forceinline__ WaveLds carve(unsigned char* base, const LdsLayout& l) {
    WaveLds L;
    L.nodes = reinterpret_cast<Node*>(base);
    L.cb = reinterpret_cast<unsigned short*>(base + l.off_cb);
    L.path = reinterpret_cast<unsigned short*>(base + l.off_path);
    L.xh = reinterpret_cast<float*>(base + l.off_xh);
    L.xa = reinterpret_cast<float*>(base + l.off_xa);
    L.xb = reinterpret_cast<float*>(base + l.off_xb);
    L.ob = reinterpret_cast<float*>(base + l.off_ob);
    L.vc = reinterpret_cast<float*>(base + l.off_vc);
    return L;
}

/* lane pair (2i, 2i+1) of a global row of length n */
__device__ __forceinline__ Pair pair_from_global(const float* row, int n, int lane) {
    Pair p;
    const int i = 2 * lane;
    p.va = i < n;
    p.vb = i + 1 < n;
    p.a = p.va ? row[i] : 0.0f;
    p.b = p.vb ? row[i + 1] : 0.0f;
    return p;
}

__device__ __forceinline__ void pair_to_global(float* row, const Pair p, int lane) {
    const int i = 2 * lane;
    if (p.va) row[i] = p.a;
    if (p.vb) row[i + 1] = p.b;
}

/* ------------------------------------------------------------------------------
 * Standalone batched inference (wave per sample): the Muzero.*_inference wrappers
 * (muzero_model.py:828-905).
 * ---------------------------------------------------------------------------- */
struct InferParams {
    Model m;
    LdsLayout lds;
    int batch;
    const float* in;       /* obs [B][obs_dim] (vision: [B][3][98][98]) or hidden [B][hid] */
    const int* action;     /* [B]                                */
    float* reward;         /* [B]                                */
    float* hidden_out;     /* [B][hid]                           */
    float* policy;         /* [B][A] (kLogits: the softmax's logits) */
    float* value;          /* [B]                                */
    long long hidden_stride; /* floats between the rows of hidden_out (0: hid) */
};

enum { kInferInitial = 0, kInferRecurrent = 1, kInferPrediction = 2 };

template <int kMode, bool kVision = false, bool kLogits = false>
__global__ void __launch_bounds__(256) k_inference(const InferParams p) {
    extern __shared__ __align__(16) unsigned char smem[];
    const int lane = lane_id();
    const int wave = threadIdx.x >> 6;
    const int b = blockIdx.x * (blockDim.x >> 6) + wave;
    if (b >= p.batch) return;
    const WaveLds L = carve(smem + (size_t)wave * p.lds.bytes, p.lds);
    const Model& m = p.m;
    constexpr bool vision = kVision;
    const size_t obs_floats = vision ? (size_t)MZS_VIS_C * m.obs_dim * m.obs_dim : (size_t)m.obs_dim;
    const int n_in = kMode == kInferInitial ? (vision ? 0 : m.obs_dim) : m.hid;
    for (int k = lane; k < n_in; k += kWave) L.xh[k] = p.in[(size_t)b * n_in + k];
    wave_sync();
    if constexpr (kVision) vis_cache_load(m.blob, vis_offsets(m), L.vc, lane);
    if (kMode == kInferInitial) {
        model_representation<kVision>(m, L, p.in + (size_t)b * obs_floats, nullptr, lane);
    } else if (kMode == kInferRecurrent) {
        const float reward = model_dynamics<kVision>(m, L, p.action[b], nullptr, lane);
        if (lane == 0) p.reward[b] = reward;
    }
    if (kMode != kInferPrediction) {
        const size_t hs = p.hidden_stride ? (size_t)p.hidden_stride : (size_t)m.hid;
        for (int k = lane; k < m.hid; k += kWave) p.hidden_out[(size_t)b * hs + k] = L.xh[k];
    }
    if (p.policy || p.value) {
        Pair pol;
        const float value = model_prediction<kVision, 64, kLogits>(m, L, &pol, lane);
        if (p.policy) pair_to_global(p.policy + (size_t)b * m.A, pol, lane);
        if (p.value && lane == 0) p.value[b] = value;
    }
}

typedef void (*infer_kernel_t)(const InferParams);
infer_kernel_t pick_logits_kernel(bool vision); /* mzs_logits.hip */

}  // namespace mzs
#endif
