// The norms around a block in one pass: r = x + scale o gate o N_post(y) (what leaves the block before) and z = N_pre(r) (what enters the
// next one), with the gradients of everything. N: LayerNorm, RMS norm or none. Both are bound by HBM: every row is read once, kept in
// registers and written once; r is normalised before it is rounded.
//
// A workgroup of ceil(D / 512) waves owns a row, eight neighbouring columns per lane. Backward, it walks the rows of one sample with four
// column sums in registers -- dR, dR o y^, dz, dz o r^ -- from which all parameter gradients follow, because gate and scale do not vary
// within a sample:
//   dgate_b = scale o sum t,  dscale = sum_b gate_b o sum t,  t = w o (dR o y^) + bias o dR;   dw_post = sum_b f_b o sum (dR o y^),
//   dbias_post = sum_b f_b o sum dR  (f_b = scale o gate_b);   dw_pre = sum dz o r^,  dbias_pre = sum dz.
// The partial sums of the workgroups are added in their order: the results do not depend on the schedule.
#include <algorithm>

#include "blocks.h"

namespace isb {
namespace {

// eight neighbouring values at p + c (c < D; VEC: D % 8 == 0 and 16-byte rows), zeros past D
template <int DT, bool VEC>
__device__ __forceinline__ void load8(const void* base, int64_t row, int c, int D, float (&v)[8]) {
    if constexpr (DT == 0) {
        const float* p = static_cast<const float*>(base) + row * D + c;
        if constexpr (VEC) {
            const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = c + i < D ? p[i] : 0.f;
        }
    } else {
        using T = T16<DT == 1>;
        const uint16_t* p = static_cast<const uint16_t*>(base) + row * D + c;
        if constexpr (VEC) {
            const uint4 a = *reinterpret_cast<const uint4*>(p);
            v[0] = T::lo(a.x); v[1] = T::hi(a.x); v[2] = T::lo(a.y); v[3] = T::hi(a.y); v[4] = T::lo(a.z); v[5] = T::hi(a.z); v[6] = T::lo(a.w); v[7] = T::hi(a.w);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = c + i < D ? T::to_f32(p[i]) : 0.f;
        }
    }
}
template <int DT, bool VEC>
__device__ __forceinline__ void store8(void* base, int64_t row, int c, int D, const float (&v)[8]) {
    if constexpr (DT == 0) {
        float* p = static_cast<float*>(base) + row * D + c;
        if constexpr (VEC) {
            *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) if (c + i < D) p[i] = v[i];
        }
    } else {
        using T = T16<DT == 1>;
        uint16_t* p = static_cast<uint16_t*>(base) + row * D + c;
        if constexpr (VEC) {
            *reinterpret_cast<uint4*>(p) = make_uint4(T::pack2(v[0], v[1]), T::pack2(v[2], v[3]), T::pack2(v[4], v[5]), T::pack2(v[6], v[7]));
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) if (c + i < D) p[i] = T::from_f32(v[i]);
        }
    }
}
__device__ __forceinline__ void param8(const float* p, int c, int D, float fill, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = p && c + i < D ? p[c + i] : fill;
}

// sums of N values over the workgroup, the same bits in every lane. The buffer's two halves take turns, so one barrier per call is enough.
template <int MOST>
struct Meet {
    float* buf;                              // [2][16 waves][MOST]
    int waves, wave, lane, slot;
    template <int N>
    __device__ __forceinline__ void sum(float (&v)[N]) {
        static_assert(N <= MOST, "buffer");
#pragma unroll
        for (int o = 32; o; o >>= 1)
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], o);
        if (waves == 1) return;
        float* s = buf + slot * 16 * MOST;
        slot ^= 1;
        if (lane == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) s[wave * MOST + i] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = 0.f;
        for (int w = 0; w < waves; ++w)
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] += s[w * MOST + i];
    }
};

// R rows v -> (v - mean) inv (RMS: no mean); columns past D stay zero. Which of the norms runs comes as separate flags: the compiler of
// ROCm 7.2 makes ONE three-way switch of tests on a single `kind` and lowers its default case (uniform, a loop around it) wrongly -- the
// copies into the merged registers are skipped.
template <int R>
__device__ __forceinline__ void normalise(bool centred, float (&v)[R][8], int c, int D, float eps, float (&mean)[R], float (&inv)[R], Meet<2 * R>& meet) {
#pragma unroll
    for (int k = 0; k < R; ++k) mean[k] = 0.f;
    if (centred) {
#pragma unroll
        for (int k = 0; k < R; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) mean[k] += v[k][i];
        meet.sum(mean);
#pragma unroll
        for (int k = 0; k < R; ++k) {
            mean[k] = mean[k] / (float)D;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[k][i] = c + i < D ? v[k][i] - mean[k] : 0.f;
        }
    }
    float s[R] = {};
#pragma unroll
    for (int k = 0; k < R; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) s[k] = __builtin_fmaf(v[k][i], v[k][i], s[k]);
    meet.sum(s);
#pragma unroll
    for (int k = 0; k < R; ++k) {
        inv[k] = 1.0f / sqrtf(s[k] / (float)D + eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[k][i] *= inv[k];
    }
}

// R rows at a time: their loads are in flight together and they share the barriers
template <int DT, bool VEC, int R, int MOST>
__global__ __launch_bounds__(MOST) void norm_fwd_kernel(NormArgs a, int64_t rows) {
    if constexpr (DT == 1) T16<true>::enter();
    __shared__ float buf[2 * 16 * 2 * R];
    const int tid = threadIdx.x, c = tid * 8, D = a.D;
    const bool in = c < D;
    Meet<2 * R> meet{buf, (int)blockDim.x >> 6, tid >> 6, tid & 63, 0};
    float qw[8], qb[8], pw[8], pb[8], sc[8];
    param8(a.post_w, c, D, 1.f, qw);
    param8(a.post_b, c, D, 0.f, qb);
    param8(a.pre_w, c, D, 1.f, pw);
    param8(a.pre_b, c, D, 0.f, pb);
    param8(a.scale, c, D, 1.f, sc);
    for (int64_t row = (int64_t)blockIdx.x * R; row < rows; row += (int64_t)gridDim.x * R) {
        const int n = (int)min((int64_t)R, rows - row);
        float r[R][8] = {}, y[R][8] = {};
#pragma unroll
        for (int k = 0; k < R; ++k)
            if (in && k < n) {
                load8<DT, VEC>(a.x, row + k, c, D, r[k]);
                if (a.y) load8<DT, VEC>(a.y, row + k, c, D, y[k]);
            }
        float my[R] = {}, iy[R], mr[R] = {}, ir[R];
#pragma unroll
        for (int k = 0; k < R; ++k) iy[k] = ir[k] = 1.f;
        if (a.y) {
            if (a.post) normalise<R>(a.post_centred, y, c, D, a.eps, my, iy, meet);
#pragma unroll
            for (int k = 0; k < R; ++k) {
                float g[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) g[i] = 1.f;
                if (a.gate && in && k < n) load8<DT, VEC>(a.gate, (row + k) / a.L, c, D, g);
#pragma unroll
                for (int i = 0; i < 8; ++i) r[k][i] = c + i < D ? __builtin_fmaf(sc[i] * g[i], __builtin_fmaf(y[k][i], qw[i], qb[i]), r[k][i]) : 0.f;
                if (in && k < n) store8<DT, VEC>(a.r, row + k, c, D, r[k]);
            }
        }
        if (a.pre) {
            normalise<R>(a.pre_centred, r, c, D, a.eps, mr, ir, meet);
#pragma unroll
            for (int k = 0; k < R; ++k) {
#pragma unroll
                for (int i = 0; i < 8; ++i) r[k][i] = __builtin_fmaf(r[k][i], pw[i], pb[i]);
                if (in && k < n) store8<DT, VEC>(a.z, row + k, c, D, r[k]);
            }
        }
        if (a.stats && tid == 0) {
#pragma unroll
            for (int k = 0; k < R; ++k)
                if (k < n) *reinterpret_cast<float4*>(a.stats + 4 * (row + k)) = make_float4(my[k], iy[k], mr[k], ir[k]);
        }
    }
}

template <int DT, bool VEC, int R, int MOST>
__global__ __launch_bounds__(MOST) void norm_bwd_kernel(NormArgs a) {
    if constexpr (DT == 1) T16<true>::enter();
    __shared__ float buf[2 * 16 * 2 * R];
    const int tid = threadIdx.x, c = tid * 8, D = a.D;
    const bool in = c < D;
    Meet<2 * R> meet{buf, (int)blockDim.x >> 6, tid >> 6, tid & 63, 0};
    const int b = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    const int l0 = chunk * a.rows_per_chunk, l1 = min(a.L, l0 + a.rows_per_chunk);
    float qw[8], qb[8], pw[8], f[8], g[8];
    param8(a.post_w, c, D, 1.f, qw);
    param8(a.post_b, c, D, 0.f, qb);
    param8(a.pre_w, c, D, 1.f, pw);
    param8(a.scale, c, D, 1.f, f);
    if (a.gate && in) {
        load8<DT, VEC>(a.gate, b, c, D, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] *= g[i];
    }
    const float rD = 1.0f / (float)D;
    float s0[8] = {}, s1[8] = {}, s2[8] = {}, s3[8] = {};
    for (int l = l0; l < l1; l += R) {
        const int64_t row = (int64_t)b * a.L + l;
        const int n = min(R, l1 - l);
        float x[R][8] = {}, y[R][8] = {}, dr[R][8] = {}, dz[R][8] = {};
        float4 st[R];
#pragma unroll
        for (int k = 0; k < R; ++k) {
            st[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (k < n) {
                if (in) {
                    load8<DT, VEC>(a.x, row + k, c, D, x[k]);
                    if (a.y) load8<DT, VEC>(a.y, row + k, c, D, y[k]);
                    if (a.dr) load8<DT, VEC>(a.dr, row + k, c, D, dr[k]);
                    if (a.pre) load8<DT, VEC>(a.dz, row + k, c, D, dz[k]);
                }
                st[k] = *reinterpret_cast<const float4*>(a.stats + 4 * (row + k));
            }
        }
        // (rows past the chunk: dr, dz and 1 / sd are zero, so they add nothing to any sum)
        if (a.y) {
#pragma unroll
            for (int k = 0; k < R; ++k)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    y[k][i] = c + i < D ? (y[k][i] - st[k].x) * st[k].y : 0.f;
                    x[k][i] = __builtin_fmaf(f[i], __builtin_fmaf(y[k][i], qw[i], qb[i]), x[k][i]);
                }
        }
        if (a.pre) {
            float t[2 * R] = {};
#pragma unroll
            for (int k = 0; k < R; ++k)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x[k][i] = c + i < D ? (x[k][i] - st[k].z) * st[k].w : 0.f;                 // r^
                    const float d = dz[k][i] * pw[i];
                    t[2 * k] += d;
                    t[2 * k + 1] = __builtin_fmaf(d, x[k][i], t[2 * k + 1]);
                    s2[i] += dz[k][i];
                    s3[i] = __builtin_fmaf(dz[k][i], x[k][i], s3[i]);
                }
            meet.sum(t);
#pragma unroll
            for (int k = 0; k < R; ++k) {
                const float m0 = a.pre_centred ? t[2 * k] * rD : 0.f, m1 = t[2 * k + 1] * rD;
#pragma unroll
                for (int i = 0; i < 8; ++i) dr[k][i] = c + i < D ? __builtin_fmaf(st[k].w, dz[k][i] * pw[i] - m0 - x[k][i] * m1, dr[k][i]) : 0.f;
            }
        }
#pragma unroll
        for (int k = 0; k < R; ++k)
            if (in && k < n) store8<DT, VEC>(a.dx, row + k, c, D, dr[k]);
        if (a.y) {
            float t[2 * R] = {};
#pragma unroll
            for (int k = 0; k < R; ++k)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    s0[i] += dr[k][i];
                    s1[i] = __builtin_fmaf(dr[k][i], y[k][i], s1[i]);
                    dr[k][i] = c + i < D ? dr[k][i] * f[i] * qw[i] : 0.f;
                    t[2 * k] += dr[k][i];
                    t[2 * k + 1] = __builtin_fmaf(dr[k][i], y[k][i], t[2 * k + 1]);
                }
            if (a.post) {
                meet.sum(t);
#pragma unroll
                for (int k = 0; k < R; ++k) {
                    const float m0 = a.post_centred ? t[2 * k] * rD : 0.f, m1 = t[2 * k + 1] * rD;
#pragma unroll
                    for (int i = 0; i < 8; ++i) dr[k][i] = st[k].y * (dr[k][i] - m0 - y[k][i] * m1);
                }
            }
#pragma unroll
            for (int k = 0; k < R; ++k)
                if (in && k < n) store8<DT, VEC>(a.dy, row + k, c, D, dr[k]);
        }
    }
    float* p = a.part + (int64_t)blockIdx.x * 4 * D;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (c + i < D) { p[c + i] = s0[i]; p[D + c + i] = s1[i]; p[2 * D + c + i] = s2[i]; p[3 * D + c + i] = s3[i]; }
}

// sums over the chunks of a sample: part [B, chunks, 4, D] -> joint [B, 4, D], and the sample's dgate. 64 columns x 4 chunk lanes.
template <int DT>
__global__ __launch_bounds__(256) void norm_join_kernel(NormArgs a, float* joint) {
    if constexpr (DT == 1) T16<true>::enter();
    __shared__ float red[4][4][64];
    const int cl = threadIdx.x & 63, kl = threadIdx.x >> 6, b = blockIdx.y, c = blockIdx.x * 64 + cl, D = a.D;
    float s[4] = {};
    if (c < D)
        for (int k = kl; k < a.chunks; k += 4) {
            const float* p = a.part + ((int64_t)b * a.chunks + k) * 4 * D + c;
#pragma unroll
            for (int j = 0; j < 4; ++j) s[j] += p[j * D];
        }
#pragma unroll
    for (int j = 0; j < 4; ++j) red[kl][j][cl] = s[j];
    __syncthreads();
    if (c >= D) return;
    joint[((int64_t)b * 4 + kl) * D + c] = red[0][kl][cl] + red[1][kl][cl] + red[2][kl][cl] + red[3][kl][cl];
    if (kl == 0 && a.dgate) {
        float t[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) t[j] = red[0][j][cl] + red[1][j][cl] + red[2][j][cl] + red[3][j][cl];
        const float w = a.post_w ? a.post_w[c] : 1.f, q = a.post_b ? a.post_b[c] : 0.f;
        const float v = (a.scale ? a.scale[c] : 1.f) * (w * t[1] + q * t[0]);
        if constexpr (DT == 0) static_cast<float*>(a.dgate)[(int64_t)b * D + c] = v;
        else static_cast<uint16_t*>(a.dgate)[(int64_t)b * D + c] = T16<DT == 1>::from_f32(v);
    }
}
// joint [B, 4, D] -> the parameters' gradients: 32 columns x 8 sample lanes
template <int DT>
__global__ __launch_bounds__(256) void norm_params_kernel(NormArgs a, const float* joint) {
    __shared__ float red[8][5][32];
    const int cl = threadIdx.x & 31, bl = threadIdx.x >> 5, c = blockIdx.x * 32 + cl, D = a.D;
    float s[5] = {};                         // dscale, dw_post, dbias_post, dw_pre, dbias_pre
    if (c < D) {
        const float w = a.post_w ? a.post_w[c] : 1.f, q = a.post_b ? a.post_b[c] : 0.f, sc = a.scale ? a.scale[c] : 1.f;
        for (int b = bl; b < a.B; b += 8) {
            const float* p = joint + (int64_t)b * 4 * D + c;
            float g = 1.f;
            if (a.gate) {
                if constexpr (DT == 0) g = static_cast<const float*>(a.gate)[(int64_t)b * D + c];
                else g = T16<DT == 1>::to_f32(static_cast<const uint16_t*>(a.gate)[(int64_t)b * D + c]);
            }
            const float a0 = p[0], a1 = p[D];
            s[0] += g * (w * a1 + q * a0);
            s[1] += sc * g * a1;
            s[2] += sc * g * a0;
            s[3] += p[3 * D];
            s[4] += p[2 * D];
        }
    }
#pragma unroll
    for (int j = 0; j < 5; ++j) red[bl][j][cl] = s[j];
    __syncthreads();
    if (c >= D || bl >= 5) return;
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) t += red[k][bl][cl];
    float* out[5] = {a.d_scale, a.d_post_w, a.d_post_b, a.d_pre_w, a.d_pre_b};
    float* o = bl == 0 ? out[0] : bl == 1 ? out[1] : bl == 2 ? out[2] : bl == 3 ? out[3] : out[4];
    if (o) o[c] = t;
}

constexpr int TEAMS = 1024;               // workgroups of the backward pass: enough to fill the chip, few enough for small partial sums

bool vec_ok(const NormArgs& a) {
    uintptr_t m = 0;
    for (const void* p : {a.x, a.y, a.gate, a.dr, a.dz, (const void*)a.r, (const void*)a.z, (const void*)a.dx, (const void*)a.dy}) m |= (uintptr_t)p;
    return a.D % 8 == 0 && m % 16 == 0;
}
// chunks of rows per sample; without a gate all rows are one sample
void plan(NormArgs& a) {
    if (!a.gate) { a.L *= a.B; a.B = 1; }
    const int want = std::max(1, TEAMS / a.B);
    a.rows_per_chunk = cdiv(a.L, std::min(want, a.L));
    a.chunks = cdiv(a.L, a.rows_per_chunk);
}
template <int DT>
int fwd(const NormArgs& a, hipStream_t st) {
    const int64_t rows = (int64_t)a.B * a.L;
    const int threads = 64 * cdiv(a.D, 512);
    if (vec_ok(a) && threads <= 512 && rows >= 4096) norm_fwd_kernel<DT, true, 4, 512><<<2048, threads, 0, st>>>(a, rows);
    else if (vec_ok(a)) norm_fwd_kernel<DT, true, 1, 1024><<<(unsigned)std::min<int64_t>(rows, 8192), threads, 0, st>>>(a, rows);
    else norm_fwd_kernel<DT, false, 1, 1024><<<(unsigned)std::min<int64_t>(rows, 8192), threads, 0, st>>>(a, rows);
    ISB_LAUNCHED("norm_fwd", st);
    return ISB_OK;
}
template <int DT>
int bwd(NormArgs a, float* ws, hipStream_t st) {
    plan(a);
    a.part = ws;
    float* joint = ws + (int64_t)a.B * a.chunks * 4 * a.D;
    const int threads = 64 * cdiv(a.D, 512);
    if (vec_ok(a) && threads <= 512) norm_bwd_kernel<DT, true, 2, 512><<<a.B * a.chunks, threads, 0, st>>>(a);
    else if (vec_ok(a)) norm_bwd_kernel<DT, true, 1, 1024><<<a.B * a.chunks, threads, 0, st>>>(a);
    else norm_bwd_kernel<DT, false, 1, 1024><<<a.B * a.chunks, threads, 0, st>>>(a);
    ISB_LAUNCHED("norm_bwd", st);
    norm_join_kernel<DT><<<dim3(cdiv(a.D, 64), a.B), 256, 0, st>>>(a, joint);
    ISB_LAUNCHED("norm_join", st);
    norm_params_kernel<DT><<<cdiv(a.D, 32), 256, 0, st>>>(a, joint);
    ISB_LAUNCHED("norm_params", st);
    return ISB_OK;
}
}  // namespace

size_t norm_workspace(const NormArgs& a0) {
    NormArgs a = a0;
    plan(a);
    return ((size_t)a.B * a.chunks + a.B) * 4 * a.D * sizeof(float);
}
int launch_norm_fwd(const NormArgs& a, int dtype, hipStream_t st) { return dtype == 0 ? fwd<0>(a, st) : dtype == 1 ? fwd<1>(a, st) : fwd<2>(a, st); }
int launch_norm_bwd(NormArgs a, int dtype, float* ws, hipStream_t st) { return dtype == 0 ? bwd<0>(a, ws, st) : dtype == 1 ? bwd<1>(a, ws, st) : bwd<2>(a, ws, st); }

}  // namespace isb
