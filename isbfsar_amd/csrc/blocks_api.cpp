// C ABI of the stand-alone layer operators (include/isbfsar.h): argument checks, workspace, device; the kernels are in xattn_kernels.hip,
// ffn_kernels.hip and norm_kernels.hip.
#include <algorithm>
#include <cmath>

#include "blocks.h"

namespace {
using namespace isb;

// the calling thread's device is `device` for the call and what it was afterwards
class OnDevice {
  public:
    int enter(int device) {
        ISB_HIP(hipGetDevice(&prev_));
        if (prev_ != device) {
            const hipError_t e = hipSetDevice(device);
            if (e != hipSuccess) (void)hipGetLastError();          // (not left for the next launch to find)
            ISB_REQUIRE(e == hipSuccess, ISB_ERR_HIP, "device %d: %s", device, hipGetErrorString(e));
            changed_ = true;
        }
        return ISB_OK;
    }
    ~OnDevice() { if (changed_) (void)hipSetDevice(prev_); }

  private:
    int prev_ = 0;
    bool changed_ = false;
};

constexpr int64_t MOST = 1 << 22;           // rows of a tile x a stride of this many elements stay within a 32-bit byte offset

int aligned(const char* what, const void* p, std::initializer_list<int64_t> strides = {}) {
    ISB_REQUIRE(p, ISB_ERR_INVALID, "%s is null", what);
    ISB_REQUIRE(reinterpret_cast<uintptr_t>(p) % 16 == 0, ISB_ERR_INVALID, "%s: %p does not lie on 16 bytes", what, p);
    for (int64_t s : strides) ISB_REQUIRE(s >= 0 && s % 8 == 0, ISB_ERR_INVALID, "%s: stride %lld is not a multiple of 8", what, (long long)s);
    return ISB_OK;
}
int room(const char* what, const void* ws, size_t bytes, size_t need) {
    ISB_REQUIRE(need == 0 || (ws && bytes >= need), ISB_ERR_INVALID, "%s: workspace of %zu bytes, %zu are needed", what, ws ? bytes : 0, need);
    ISB_REQUIRE(reinterpret_cast<uintptr_t>(ws) % 16 == 0, ISB_ERR_INVALID, "%s: workspace %p does not lie on 16 bytes", what, ws);
    return ISB_OK;
}
int two_byte(const char* what, int dtype) {
    ISB_REQUIRE(dtype == ISB_T_F16 || dtype == ISB_T_BF16, ISB_ERR_INVALID, "%s: type %d is neither ISB_T_F16 nor ISB_T_BF16", what, dtype);
    return ISB_OK;
}

// ---------------------------------------------------------------- cross attention
int xattn_shape(const isb_xattn_args* u, XattnArgs& a) {
    ISB_REQUIRE(u, ISB_ERR_INVALID, "null argument");
    ISB_TRY(two_byte("cross attention", u->dtype));
    ISB_REQUIRE(u->B >= 1 && u->Bk >= 1 && u->Lq >= 1 && u->Lk >= 1 && u->Hq >= 1 && u->Hk >= 1, ISB_ERR_INVALID,
                "cross attention: bad shape B=%d Bk=%d Lq=%d Lk=%d Hq=%d Hk=%d", u->B, u->Bk, u->Lq, u->Lk, u->Hq, u->Hk);
    ISB_REQUIRE(u->D >= 8 && u->D <= 128 && u->D % 8 == 0, ISB_ERR_INVALID, "cross attention: head size %d is not a multiple of 8 up to 128", u->D);
    ISB_REQUIRE(u->B % u->Bk == 0, ISB_ERR_INVALID, "cross attention: %d samples do not share %d sets of states evenly", u->B, u->Bk);
    ISB_REQUIRE(u->Hq % u->Hk == 0, ISB_ERR_INVALID, "cross attention: %d query heads do not share %d state heads evenly", u->Hq, u->Hk);
    ISB_REQUIRE(u->Lk <= (1 << 30), ISB_ERR_INVALID, "cross attention: %d states are too many", u->Lk);
    const int64_t m = (int64_t)(u->B / u->Bk) * u->Lq * (u->Hq / u->Hk);
    ISB_REQUIRE(m <= (1 << 30), ISB_ERR_INVALID, "cross attention: %lld rows share one set of states: too many", (long long)m);
    const int64_t rows = m * u->Bk * u->Hk, states = (int64_t)u->Bk * u->Hk * u->Lk;
    ISB_REQUIRE(rows < (1ll << 31) && states < (1ll << 31), ISB_ERR_INVALID, "cross attention: %lld rows, %lld states are too many", (long long)rows,
                (long long)states);
    // (a launch holds fewer than 2^32 threads: not quite 2^23 workgroups of at most 512, their number rounded up to the 8 XCDs; splits come only
    // where there are less than 2^10)
    const int64_t groups = (int64_t)u->Bk * u->Hk, tiles = groups * std::max((m + 127) / 128, ((int64_t)u->Lk + 127) / 128);
    ISB_REQUIRE(tiles <= (1 << 23) - 8, ISB_ERR_INVALID, "cross attention: %lld tiles of 128 rows or states are more than one launch holds", (long long)tiles);
    ISB_REQUIRE(std::isfinite(u->scale) && u->scale > 0, ISB_ERR_INVALID, "cross attention: scale %g is not positive", (double)u->scale);
    a.B = u->B; a.Bk = u->Bk; a.nb = u->B / u->Bk; a.Lq = u->Lq; a.Lk = u->Lk; a.Hq = u->Hq; a.Hk = u->Hk; a.G = u->Hq / u->Hk; a.D = u->D;
    a.M = (int)m;
    a.by_lqg = FastDiv((uint32_t)(a.Lq * a.G));
    a.by_g = FastDiv((uint32_t)a.G);
    a.scale = u->scale;
    a.c = u->scale * LOG2E;
    return ISB_OK;
}
int xattn_args(const isb_xattn_args* u, bool backward, XattnArgs& a) {
    ISB_TRY(xattn_shape(u, a));
    ISB_TRY(aligned("q", u->q, {u->q_stride[0], u->q_stride[1], u->q_stride[2]}));
    ISB_TRY(aligned("k", u->k, {u->k_stride[0], u->k_stride[1], u->k_stride[2]}));
    ISB_TRY(aligned("v", u->v, {u->v_stride[0], u->v_stride[1], u->v_stride[2]}));
    ISB_REQUIRE(u->k_stride[1] <= MOST && u->v_stride[1] <= MOST, ISB_ERR_INVALID, "cross attention: the states' stride is more than %lld elements",
                (long long)MOST);
    ISB_TRY(aligned("out", u->out));
    ISB_REQUIRE(u->lse, ISB_ERR_INVALID, "lse is null");
    ISB_REQUIRE(!u->key_mask || u->mask_stride >= 0, ISB_ERR_INVALID, "key_mask: stride %lld", (long long)u->mask_stride);
    a.q = (const uint16_t*)u->q; a.k = (const uint16_t*)u->k; a.v = (const uint16_t*)u->v;
    a.q_sb = u->q_stride[0]; a.q_sl = u->q_stride[1]; a.q_sh = u->q_stride[2];
    a.k_sb = u->k_stride[0]; a.k_sl = u->k_stride[1]; a.k_sh = u->k_stride[2];
    a.v_sb = u->v_stride[0]; a.v_sl = u->v_stride[1]; a.v_sh = u->v_stride[2];
    a.kv_len = u->kv_len; a.mask = u->key_mask; a.mask_sb = u->mask_stride;
    a.out = (uint16_t*)u->out; a.lse = u->lse;
    if (backward) {
        ISB_TRY(aligned("dout", u->dout, {u->dout_stride[0], u->dout_stride[1], u->dout_stride[2]}));
        ISB_TRY(aligned("dq", u->dq));
        ISB_TRY(aligned("dk", u->dk));
        ISB_TRY(aligned("dv", u->dv));
        a.dout = (const uint16_t*)u->dout;
        a.d_sb = u->dout_stride[0]; a.d_sl = u->dout_stride[1]; a.d_sh = u->dout_stride[2];
        a.dq = (uint16_t*)u->dq; a.dk = (uint16_t*)u->dk; a.dv = (uint16_t*)u->dv;
    }
    return ISB_OK;
}
int xattn_run(const isb_xattn_args* u, bool backward, void* ws, size_t bytes, void* stream) {
    XattnArgs a{};
    ISB_TRY(xattn_args(u, backward, a));
    ISB_TRY(room("cross attention", ws, bytes, xattn_workspace(a, backward)));
    OnDevice dev;
    ISB_TRY(dev.enter(u->device));
    const bool f16 = u->dtype == ISB_T_F16;
    return backward ? launch_xattn_bwd(a, f16, (float*)ws, (hipStream_t)stream) : launch_xattn_fwd(a, f16, (float*)ws, (hipStream_t)stream);
}

// ---------------------------------------------------------------- gated feed-forward block
int ffn_shape(const isb_ffn_args* u, FfnArgs& a) {
    ISB_REQUIRE(u, ISB_ERR_INVALID, "null argument");
    ISB_TRY(two_byte("gated feed-forward", u->dtype));
    ISB_REQUIRE(u->M >= 1 && u->M <= MOST && u->D >= 8 && u->F >= 8 && u->D % 8 == 0 && u->F % 8 == 0 && u->D <= (1 << 20) && u->F <= (1 << 20),
                ISB_ERR_INVALID, "gated feed-forward: bad shape M=%d D=%d F=%d (D, F: multiples of 8)", u->M, u->D, u->F);
    ISB_REQUIRE(u->act >= ISB_ACT_SILU && u->act <= ISB_ACT_SIGMOID, ISB_ERR_INVALID, "gated feed-forward: activation %d", u->act);
    a.M = u->M; a.D = u->D; a.F = u->F; a.act = u->act;
    a.h = (uint16_t*)u->hidden;
    a.dbg = (uint16_t*)u->db_gate; a.dbu = (uint16_t*)u->db_up; a.dbd = (uint16_t*)u->db_down;
    return ISB_OK;
}
int ffn_args(const isb_ffn_args* u, bool backward, FfnArgs& a) {
    ISB_TRY(ffn_shape(u, a));
    ISB_TRY(aligned("x", u->x, {u->x_stride}));
    ISB_REQUIRE(u->M == 1 || (u->x_stride >= u->D && u->x_stride <= MOST), ISB_ERR_INVALID, "x: row stride %lld", (long long)u->x_stride);
    ISB_TRY(aligned("w_gate", u->w_gate));
    ISB_TRY(aligned("w_up", u->w_up));
    ISB_TRY(aligned("w_down", u->w_down));
    a.x = (const uint16_t*)u->x; a.x_s = u->M == 1 ? u->D : u->x_stride;
    a.wg = (const uint16_t*)u->w_gate; a.wu = (const uint16_t*)u->w_up; a.wd = (const uint16_t*)u->w_down;
    a.g = u->pre_gate; a.u = u->pre_up;
    if (!backward) {
        ISB_TRY(aligned("y", u->y));
        for (const void* b : {u->b_gate, u->b_up, u->b_down}) if (b) ISB_TRY(aligned("bias", b));
        ISB_REQUIRE((u->pre_gate == nullptr) == (u->pre_up == nullptr), ISB_ERR_INVALID, "pre_gate and pre_up: both or neither");
        if (u->pre_gate) {
            ISB_TRY(aligned("pre_gate", u->pre_gate));
            ISB_TRY(aligned("pre_up", u->pre_up));
            ISB_REQUIRE(u->hidden, ISB_ERR_INVALID, "pre_gate and pre_up need hidden too");
        }
        if (u->hidden) ISB_TRY(aligned("hidden", u->hidden));
        a.bg = (const uint16_t*)u->b_gate; a.bu = (const uint16_t*)u->b_up; a.bd = (const uint16_t*)u->b_down;
        a.y = (uint16_t*)u->y;
        return ISB_OK;
    }
    ISB_TRY(aligned("dy", u->dy, {u->dy_stride}));
    ISB_REQUIRE(u->M == 1 || (u->dy_stride >= u->D && u->dy_stride <= MOST), ISB_ERR_INVALID, "dy: row stride %lld", (long long)u->dy_stride);
    ISB_TRY(aligned("pre_gate", u->pre_gate));
    ISB_TRY(aligned("pre_up", u->pre_up));
    ISB_TRY(aligned("hidden", u->hidden));
    ISB_TRY(aligned("dx", u->dx));
    ISB_TRY(aligned("dw_gate_up", u->dw_gate_up));
    ISB_TRY(aligned("dw_down", u->dw_down));
    ISB_REQUIRE((u->db_gate == nullptr) == (u->db_up == nullptr), ISB_ERR_INVALID, "db_gate and db_up: both or neither");
    for (const void* b : {(const void*)u->db_gate, (const void*)u->db_up, (const void*)u->db_down}) if (b) ISB_TRY(aligned("bias gradient", b));
    a.dy = (const uint16_t*)u->dy; a.dy_s = u->M == 1 ? u->D : u->dy_stride;
    a.dx = (uint16_t*)u->dx; a.dwgu = (uint16_t*)u->dw_gate_up; a.dwd = (uint16_t*)u->dw_down;
    return ISB_OK;
}
int ffn_run(const isb_ffn_args* u, bool backward, void* ws, size_t bytes, void* stream) {
    FfnArgs a{};
    ISB_TRY(ffn_args(u, backward, a));
    ISB_TRY(room("gated feed-forward", ws, bytes, ffn_workspace(a, u->dtype == ISB_T_F16, backward)));
    OnDevice dev;
    ISB_TRY(dev.enter(u->device));
    const bool f16 = u->dtype == ISB_T_F16;
    return backward ? launch_ffn_bwd(a, f16, (unsigned char*)ws, (hipStream_t)stream) : launch_ffn_fwd(a, f16, (unsigned char*)ws, (hipStream_t)stream);
}

// ---------------------------------------------------------------- norms around a block
int norm_shape(const isb_norm_args* u, NormArgs& a) {
    ISB_REQUIRE(u, ISB_ERR_INVALID, "null argument");
    ISB_REQUIRE(u->dtype >= ISB_T_F32 && u->dtype <= ISB_T_BF16, ISB_ERR_INVALID, "block norm: type %d", u->dtype);
    ISB_REQUIRE(u->B >= 1 && u->L >= 1 && (int64_t)u->B * u->L <= (1 << 30) && u->D >= 1 && u->D <= 8192, ISB_ERR_INVALID,
                "block norm: bad shape B=%d L=%d D=%d (D at most 8192)", u->B, u->L, u->D);
    ISB_REQUIRE(!u->gate || u->B <= 65535, ISB_ERR_INVALID, "block norm: %d gates are too many", u->B);
    ISB_REQUIRE(u->post >= 0 && u->post <= 2 && u->pre >= 0 && u->pre <= 2, ISB_ERR_INVALID, "block norm: kinds %d, %d", u->post, u->pre);
    ISB_REQUIRE(u->y || u->pre, ISB_ERR_INVALID, "block norm: neither a block's output nor a norm: nothing to compute");
    ISB_REQUIRE(u->y || (!u->post && !u->gate && !u->scale), ISB_ERR_INVALID, "block norm: a post norm, gate or scale needs y");
    ISB_REQUIRE((u->post || !u->post_weight) && (u->post == ISB_NORM_LAYER || !u->post_bias) && (u->pre || !u->pre_weight) &&
                    (u->pre == ISB_NORM_LAYER || !u->pre_bias),
                ISB_ERR_INVALID, "block norm: a weight needs its norm, a bias a LayerNorm");
    ISB_REQUIRE(std::isfinite(u->eps) && u->eps >= 0, ISB_ERR_INVALID, "block norm: eps %g", (double)u->eps);
    a.B = u->B; a.L = u->L; a.D = u->D; a.eps = u->eps;
    a.post = u->post != ISB_NORM_NONE; a.post_centred = u->post == ISB_NORM_LAYER;
    a.pre = u->pre != ISB_NORM_NONE; a.pre_centred = u->pre == ISB_NORM_LAYER;
    a.x = u->x; a.y = u->y; a.gate = u->gate;
    a.scale = u->scale; a.post_w = u->post_weight; a.post_b = u->post_bias; a.pre_w = u->pre_weight; a.pre_b = u->pre_bias;
    a.stats = u->stats;
    const uintptr_t item = u->dtype == ISB_T_F32 ? 4 : 2;
    for (const void* p : {u->x, u->y, u->gate, (const void*)u->r, (const void*)u->z, u->dr, u->dz, (const void*)u->dx, (const void*)u->dy})
        ISB_REQUIRE(reinterpret_cast<uintptr_t>(p) % item == 0, ISB_ERR_INVALID, "block norm: %p does not lie on its type's size", p);
    ISB_REQUIRE(reinterpret_cast<uintptr_t>(u->stats) % 16 == 0, ISB_ERR_INVALID, "block norm: stats do not lie on 16 bytes");
    return ISB_OK;
}
}  // namespace

extern "C" int isb_xattn_workspace(const isb_xattn_args* u, int32_t backward, size_t* bytes) {
    return isb::guard([&]() -> int {
        ISB_REQUIRE(bytes, ISB_ERR_INVALID, "null argument");
        isb::XattnArgs a{};
        ISB_TRY(xattn_shape(u, a));
        *bytes = isb::xattn_workspace(a, backward != 0);
        return ISB_OK;
    });
}
extern "C" int isb_xattn_forward(const isb_xattn_args* a, void* ws, size_t bytes, void* stream) {
    return isb::guard([&]() -> int { return xattn_run(a, false, ws, bytes, stream); });
}
extern "C" int isb_xattn_backward(const isb_xattn_args* a, void* ws, size_t bytes, void* stream) {
    return isb::guard([&]() -> int { return xattn_run(a, true, ws, bytes, stream); });
}

extern "C" int isb_ffn_workspace(const isb_ffn_args* u, int32_t backward, size_t* bytes) {
    return isb::guard([&]() -> int {
        ISB_REQUIRE(bytes, ISB_ERR_INVALID, "null argument");
        isb::FfnArgs a{};
        ISB_TRY(ffn_shape(u, a));
        *bytes = isb::ffn_workspace(a, u->dtype == ISB_T_F16, backward != 0);
        return ISB_OK;
    });
}
extern "C" int isb_ffn_forward(const isb_ffn_args* a, void* ws, size_t bytes, void* stream) {
    return isb::guard([&]() -> int { return ffn_run(a, false, ws, bytes, stream); });
}
extern "C" int isb_ffn_backward(const isb_ffn_args* a, void* ws, size_t bytes, void* stream) {
    return isb::guard([&]() -> int { return ffn_run(a, true, ws, bytes, stream); });
}

extern "C" int isb_norm_workspace(const isb_norm_args* u, size_t* bytes) {
    return isb::guard([&]() -> int {
        ISB_REQUIRE(bytes, ISB_ERR_INVALID, "null argument");
        isb::NormArgs a{};
        ISB_TRY(norm_shape(u, a));
        *bytes = isb::norm_workspace(a);
        return ISB_OK;
    });
}
extern "C" int isb_norm_forward(const isb_norm_args* u, void* stream) {
    return isb::guard([&]() -> int {
        isb::NormArgs a{};
        ISB_TRY(norm_shape(u, a));
        ISB_REQUIRE(u->x && (!u->y || u->r) && (!u->pre || u->z), ISB_ERR_INVALID, "block norm: null argument");
        a.r = u->r;
        a.z = u->z;
        OnDevice dev;
        ISB_TRY(dev.enter(u->device));
        return isb::launch_norm_fwd(a, u->dtype, (hipStream_t)stream);
    });
}
extern "C" int isb_norm_backward(const isb_norm_args* u, void* ws, size_t bytes, void* stream) {
    return isb::guard([&]() -> int {
        isb::NormArgs a{};
        ISB_TRY(norm_shape(u, a));
        ISB_REQUIRE(u->x && u->stats && u->dx && (!u->y || u->dy) && (u->pre ? u->dz != nullptr : u->dr != nullptr), ISB_ERR_INVALID,
                    "block norm: null argument");
        ISB_REQUIRE(!u->dgate || u->gate, ISB_ERR_INVALID, "block norm: dgate without a gate");
        ISB_TRY(room("block norm", ws, bytes, isb::norm_workspace(a)));
        a.dr = u->dr; a.dz = u->dz; a.dx = u->dx; a.dy = u->dy; a.dgate = u->dgate;
        a.d_scale = u->dscale; a.d_post_w = u->dpost_weight; a.d_post_b = u->dpost_bias; a.d_pre_w = u->dpre_weight; a.d_pre_b = u->dpre_bias;
        OnDevice dev;
        ISB_TRY(dev.enter(u->device));
        return isb::launch_norm_bwd(a, u->dtype, (float*)ws, (hipStream_t)stream);
    });
}
