// Argument blocks + host launchers of the stand-alone layer operators, shared by their translation units and blocks_api.cpp.
#pragma once
#include <atomic>

#include "blk_common.h"

namespace isb {

// Kernel may use `bytes` (always the same) of dynamic LDS on the current device: asked of the runtime once per device. The operators have no
// handle, so threads that drive different devices meet here.
template <auto Kernel>
int allow_lds(size_t bytes) {
    static std::atomic<uint64_t> done{0};                // a bit per device
    int dev = 0;
    ISB_HIP(hipGetDevice(&dev));
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (done.load(std::memory_order_acquire) & bit) return ISB_OK;
    ISB_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(Kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    done.fetch_or(bit, std::memory_order_release);
    return ISB_OK;
}

// ---------------------------------------------------------------- xattn_kernels.hip
// Rows: every query row that reads the same states (bk, hk) -- the nb = B / Bk samples that share them, Lq positions, G = Hq / Hk heads --
// forms ONE list of M = nb Lq G rows (row r: sample r / (Lq G), position (r / G) % Lq, head r % G). A tile of rows is then full also for
// single tokens with grouped heads, and the gradients of shared heads and shared states are plain sums over the list.
struct XattnArgs {
    const uint16_t *q, *k, *v, *dout;                    // strides in elements, innermost dimension contiguous
    int64_t q_sb, q_sl, q_sh, k_sb, k_sl, k_sh, v_sb, v_sl, v_sh, d_sb, d_sl, d_sh;
    const int32_t* kv_len;                               // [Bk] or null
    const uint8_t* mask;                                 // [Bk, Lk] (row stride mask_sb) or null; 0 = masked
    int64_t mask_sb;
    uint16_t* out;                                       // [B, Lq, Hq, D]
    float* lse;                                          // [B, Hq, Lq]
    uint16_t *dq, *dk, *dv;                              // contiguous, shapes of q, k, v
    float* delta;                                        // backward: [Bk, Hk, M] rowsum(dout * out)
    uint16_t* zeros;                                     // 16 bytes of zeros
    float* part;                                         // partial results of the splits
    float* part2;
    FastDiv by_lqg, by_g;
    int B, Bk, nb, Lq, Lk, Hq, Hk, G, D, M;
    int n_items;                                         // work items of the launch
    int tiles, splits, chunk;                            // row (or key) tiles per group, splits of the long axis, its keys (rows) per split
    int walk;                                            // rows can be stepped through (RowWalk)
    float c, scale;                                      // scale * log2(e), scale
};
size_t xattn_workspace(const XattnArgs& a, bool backward);
int launch_xattn_fwd(XattnArgs a, bool f16, float* ws, hipStream_t st);
int launch_xattn_bwd(XattnArgs a, bool f16, float* ws, hipStream_t st);

// ---------------------------------------------------------------- ffn_kernels.hip
struct FfnArgs {
    const uint16_t *x, *wg, *wu, *wd, *bg, *bu, *bd;     // x [M, D] (row stride x_s), w_gate / w_up [F, D], w_down [D, F], biases or null
    int64_t x_s;
    uint16_t* y;                                         // [M, D]
    float *g, *u;                                        // saved pre-activations [M, F] or null
    uint16_t* h;                                         // [M, F]
    const uint16_t* dy;                                  // [M, D] (row stride dy_s)
    int64_t dy_s;
    uint16_t *dgu;                                       // [M, 2 F] workspace
    uint16_t *dx, *dwgu, *dwd, *dbg, *dbu, *dbd;         // dwgu [2 F, D]
    int M, D, F, act;
};
size_t ffn_workspace(const FfnArgs& a, bool f16, bool backward);
int launch_ffn_fwd(const FfnArgs& a, bool f16, unsigned char* ws, hipStream_t st);
int launch_ffn_bwd(const FfnArgs& a, bool f16, unsigned char* ws, hipStream_t st);

// ---------------------------------------------------------------- norm_kernels.hip
struct NormArgs {
    const void *x, *y, *gate, *dr, *dz;                  // [B, L, D] contiguous; gate [B, D]
    const float *scale, *post_w, *post_b, *pre_w, *pre_b;
    void *r, *z, *dx, *dy;
    void* dgate;
    float* stats;                                        // [B L, 4]: mean, 1 / sd of y; mean, 1 / sd of r
    float *d_scale, *d_post_w, *d_post_b, *d_pre_w, *d_pre_b;
    float* part;                                         // [B, chunks, 4, D]
    int B, L, D, chunks, rows_per_chunk;
    int post, post_centred, pre, pre_centred;            // is there a norm; does it take the mean off (LayerNorm)
    float eps;
};
size_t norm_workspace(const NormArgs& a);
int launch_norm_fwd(const NormArgs& a, int dtype, hipStream_t st);
int launch_norm_bwd(NormArgs a, int dtype, float* ws, hipStream_t st);

}  // namespace isb
