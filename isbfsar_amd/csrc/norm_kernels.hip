// The norms around a block in one pass: r = x + scale o gate o N_post(y) (what leaves the block before) and z = N_pre(r) (what enters the
// next one), with the gradients of everything. N: LayerNorm, RMS norm or none. Both are bound by HBM: every row is read once, kept in
// registers and written once; r is normalised before it is rounded. 32704 rows of 1280, bf16: forward 81 us (4.1 TB/s), backward 120 us
// (4.2 TB/s), the two small launches behind it 11. Widths that are no multiple of 8 are read a value at a time: 1279 instead of 1280 forward 242,
// backward 411 us (f32 390, 684).
//
// A workgroup of ceil(D / 512) waves owns a row, eight neighbouring columns per lane. Backward, it walks the rows of one sample with four
// column sums in registers -- dR, dR o y^, dz, dz o r^ -- from which all parameter gradients follow, because gate and scale do not vary
// within a sample:
//   dgate_b = scale o sum t,  dscale = sum_b gate_b o sum t,  t = w o (dR o y^) + bias o dR;   dw_post = sum_b f_b o sum (dR o y^),
//   dbias_post = sum_b f_b o sum dR  (f_b = scale o gate_b);   dw_pre = sum dz o r^,  dbias_pre = sum dz.
// The partial sums of the workgroups are added in their order: the results do not depend on the schedule. With many short samples
// (MANY, `plan`) a workgroup walks several whole ones, writes their dgate itself and adds sum dR and sum dR o y^ up with each sample's gate: the partial sums
// are then as many as the workgroups, not the samples, and the gate is done with (65535 samples of one row of 8192: 136 MB for 17 GB).
#include <algorithm>

#include "blocks.h"

namespace isb {
namespace {

// eight neighbouring values of a row at column c, as they lie in memory (VEC: D % 8 == 0 and 16-byte rows; else zeros past D): a row is
// requested one row ahead and unpacked when its turn comes
template <int DT, bool VEC>
struct Row8 {
    uint4 a = make_uint4(0, 0, 0, 0), b = make_uint4(0, 0, 0, 0);            // b: f32's second half
    __device__ __forceinline__ void load(const void* base, int64_t row, int c, int D) {
        if constexpr (DT == 0) {
            const uint32_t* p = static_cast<const uint32_t*>(base) + row * D + c;
            if constexpr (VEC) {
                a = reinterpret_cast<const uint4*>(p)[0];
                b = reinterpret_cast<const uint4*>(p)[1];
            } else {
                uint32_t w[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = c + i < D ? p[i] : 0u;
                a = make_uint4(w[0], w[1], w[2], w[3]);
                b = make_uint4(w[4], w[5], w[6], w[7]);
            }
        } else {
            const uint16_t* p = static_cast<const uint16_t*>(base) + row * D + c;
            if constexpr (VEC) {
                a = *reinterpret_cast<const uint4*>(p);
            } else {
                uint32_t w[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = c + i < D ? p[i] : 0u;
                a = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
            }
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        if constexpr (DT == 0) {
            v[0] = __uint_as_float(a.x); v[1] = __uint_as_float(a.y); v[2] = __uint_as_float(a.z); v[3] = __uint_as_float(a.w);
            v[4] = __uint_as_float(b.x); v[5] = __uint_as_float(b.y); v[6] = __uint_as_float(b.z); v[7] = __uint_as_float(b.w);
        } else {
            using T = T16<DT == 1>;
            v[0] = T::lo(a.x); v[1] = T::hi(a.x); v[2] = T::lo(a.y); v[3] = T::hi(a.y);
            v[4] = T::lo(a.z); v[5] = T::hi(a.z); v[6] = T::lo(a.w); v[7] = T::hi(a.w);
        }
    }
};
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

// sum over the 64 lanes, in every lane, on the vector ALU alone (lane exchanges of 1, 2, 4, 8 as DPP, of 16 and 32 as row swaps)
__device__ __forceinline__ float lanes_sum(float v) {
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xf, 0xf, true));      // quad_perm 1 0 3 2
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xf, 0xf, true));      // quad_perm 2 3 0 1
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xf, 0xf, true));     // half a row mirrored
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xf, 0xf, true));     // a row of 16 mirrored
    const u32x2 r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return sum_halves(__uint_as_float(r.x) + __uint_as_float(r.y));
}

// sums over the workgroup, the same bits in every lane. The buffer's two halves take turns, so one barrier per call is enough.
struct Meet {
    float* buf;                              // [2][16 waves][2]
    int waves, wave, lane, slot;
    __device__ __forceinline__ void sum2(float& a, float& b) {
        a = lanes_sum(a);
        b = lanes_sum(b);
        if (waves == 1) return;
        float* s = buf + slot * 32;
        slot ^= 1;
        if (lane == 0) *reinterpret_cast<float2*>(s + 2 * wave) = make_float2(a, b);
        __syncthreads();
        a = b = 0.f;
        for (int w = 0; w < waves; ++w) {
            const float2 t = *reinterpret_cast<const float2*>(s + 2 * w);
            a += t.x;
            b += t.y;
        }
    }
    __device__ __forceinline__ float sum(float a) {
        a = lanes_sum(a);
        if (waves == 1) return a;
        float* s = buf + slot * 32;
        slot ^= 1;
        if (lane == 0) s[wave] = a;
        __syncthreads();
        a = 0.f;
        for (int w = 0; w < waves; ++w) a += s[w];
        return a;
    }
};

// v -> (v - mean) inv (RMS: no mean); columns past D stay zero. Which of the norms runs comes as separate flags: the compiler of ROCm 7.2
// makes ONE three-way switch of tests on a single `kind` and lowers its default case (uniform, a loop around it) wrongly -- the copies into
// the merged registers are skipped.
__device__ __forceinline__ void normalise(bool centred, float (&v)[8], int c, int D, float eps, float& mean, float& inv, Meet& meet) {
    mean = 0.f;
    if (centred) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += v[i];
        mean = meet.sum(s) / (float)D;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < D ? v[i] - mean : 0.f;
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s = __builtin_fmaf(v[i], v[i], s);
    inv = 1.0f / sqrtf(meet.sum(s) / (float)D + eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= inv;
}

template <int DT, bool VEC, int MOST>
__global__ __launch_bounds__(MOST, MOST <= 256 ? 5 : 4) void norm_fwd_kernel(NormArgs a, int rows) {
    if constexpr (DT == 1) T16<true>::enter();
    __shared__ __attribute__((aligned(16))) float buf[64];
    const int tid = threadIdx.x, c = tid * 8, D = a.D;
    const bool in = c < D;
    Meet meet{buf, (int)blockDim.x >> 6, tid >> 6, tid & 63, 0};
    float qw[8], qb[8], pw[8], pb[8];
    param8(a.post_w, c, D, 1.f, qw);
    param8(a.post_b, c, D, 0.f, qb);
    param8(a.pre_w, c, D, 1.f, pw);
    param8(a.pre_b, c, D, 0.f, pb);
    if (a.scale) {
        float sc[8];
        param8(a.scale, c, D, 1.f, sc);
#pragma unroll
        for (int i = 0; i < 8; ++i) { qw[i] *= sc[i]; qb[i] *= sc[i]; }
    }
    Row8<DT, VEC> nx, ny;
    auto request = [&](int row) {
        if (in && row < rows) {
            nx.load(a.x, row, c, D);
            if (a.y) ny.load(a.y, row, c, D);
        }
    };
    request(blockIdx.x);
    for (int row = blockIdx.x; row < rows; row += gridDim.x) {
        float r[8], y[8], g[8];
        nx.get(r);
        ny.get(y);
        request(row + gridDim.x);
        float my = 0.f, iy = 1.f, mr = 0.f, ir = 1.f;
        if (a.y) {
#pragma unroll
            for (int i = 0; i < 8; ++i) g[i] = 1.f;
            if (a.gate && in) {
                Row8<DT, VEC> t;
                t.load(a.gate, row / a.L, c, D);
                t.get(g);
            }
            if (a.post) normalise(a.post_centred, y, c, D, a.eps, my, iy, meet);
#pragma unroll
            for (int i = 0; i < 8; ++i) r[i] = c + i < D ? __builtin_fmaf(g[i], __builtin_fmaf(y[i], qw[i], qb[i]), r[i]) : 0.f;
            if (in) store8<DT, VEC>(a.r, row, c, D, r);
        }
        if (a.pre) {
            normalise(a.pre_centred, r, c, D, a.eps, mr, ir, meet);
#pragma unroll
            for (int i = 0; i < 8; ++i) r[i] = __builtin_fmaf(r[i], pw[i], pb[i]);
            if (in) store8<DT, VEC>(a.z, row, c, D, r);
        }
        if (a.stats && tid == 0) *reinterpret_cast<float4*>(a.stats + 4 * (int64_t)row) = make_float4(my, iy, mr, ir);
    }
}

template <int DT, bool VEC, int MOST, bool MANY>
__global__ __launch_bounds__(MOST, MOST <= 256 ? 3 : 4) void norm_bwd_kernel(NormArgs a) {
    if constexpr (DT == 1) T16<true>::enter();
    __shared__ __attribute__((aligned(16))) float buf[64];
    const int tid = threadIdx.x, c = tid * 8, D = a.D;
    const bool in = c < D;
    Meet meet{buf, (int)blockDim.x >> 6, tid >> 6, tid & 63, 0};
    // a chunk of one sample's rows, or (MANY: rows_per_chunk counts samples) the rows of several whole samples
    const int chunk = blockIdx.x % a.chunks, b0 = MANY ? chunk * a.rows_per_chunk : blockIdx.x / a.chunks;
    const int l0 = MANY ? 0 : chunk * a.rows_per_chunk, l1 = MANY ? (min(a.B, b0 + a.rows_per_chunk) - b0) * a.L : min(a.L, l0 + a.rows_per_chunk);
    int b = b0, end = a.L;                                    // MANY: the sample, the row behind its last
    float qw[8], qb[8], pw[8], f[8];
    param8(a.post_w, c, D, 1.f, qw);
    param8(a.post_b, c, D, 0.f, qb);
    param8(a.pre_w, c, D, 1.f, pw);
    param8(a.scale, c, D, 1.f, f);
    Row8<DT, VEC> gate, ng;                                   // this sample's, the next one's (MANY)
    if (a.gate && in) {
        float g[8];
        gate.load(a.gate, b, c, D);
        gate.get(g);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] *= g[i];
    }
    const float rD = 1.0f / (float)D;
    float s0[8] = {}, s1[8] = {}, s2[8] = {}, s3[8] = {};
    // MANY: s0 and s1 with the gates, over the samples; every lane its own (registers are taken)
    __shared__ float all[MANY ? 16 * MOST : 1];
    if (MANY) {
#pragma unroll
        for (int i = 0; i < 16; ++i) all[i * MOST + tid] = 0.f;
    }
    Row8<DT, VEC> nx, ny, ndr, ndz;
    float4 nst = make_float4(0.f, 0.f, 0.f, 0.f);
    auto request = [&](int l, bool next_sample) {
        if (l >= l1) return;
        const int64_t row = (int64_t)b0 * a.L + l;
        if (in) {
            if (MANY && next_sample) ng.load(a.gate, b + 1, c, D);
            nx.load(a.x, row, c, D);
            if (a.y) ny.load(a.y, row, c, D);
            if (a.dr) ndr.load(a.dr, row, c, D);
            if (a.pre) ndz.load(a.dz, row, c, D);
        }
        nst = *reinterpret_cast<const float4*>(a.stats + 4 * row);
    };
    request(l0, false);
    for (int l = l0; l < l1; ++l) {
        const int64_t row = (int64_t)b0 * a.L + l;
        float x[8], y[8], dr[8], dz[8];
        nx.get(x);
        ny.get(y);
        ndr.get(dr);
        ndz.get(dz);
        const float4 st = nst;
        const bool ends = MANY && l + 1 == end;
        request(l + 1, ends);
        if (a.y) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                y[i] = c + i < D ? (y[i] - st.x) * st.y : 0.f;
                x[i] = __builtin_fmaf(f[i], __builtin_fmaf(y[i], qw[i], qb[i]), x[i]);
            }
        }
        if (a.pre) {
            float t0 = 0.f, t1 = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = c + i < D ? (x[i] - st.z) * st.w : 0.f;                 // r^
                const float d = dz[i] * pw[i];
                t0 += d;
                t1 = __builtin_fmaf(d, x[i], t1);
                s2[i] += dz[i];
                s3[i] = __builtin_fmaf(dz[i], x[i], s3[i]);
            }
            meet.sum2(t0, t1);
            const float m0 = a.pre_centred ? t0 * rD : 0.f, m1 = t1 * rD;
#pragma unroll
            for (int i = 0; i < 8; ++i) dr[i] = c + i < D ? __builtin_fmaf(st.w, dz[i] * pw[i] - m0 - x[i] * m1, dr[i]) : 0.f;
        }
        if (in) store8<DT, VEC>(a.dx, row, c, D, dr);
        if (a.y) {
            float t0 = 0.f, t1 = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                s0[i] += dr[i];
                s1[i] = __builtin_fmaf(dr[i], y[i], s1[i]);
                dr[i] = c + i < D ? dr[i] * f[i] * qw[i] : 0.f;
                t0 += dr[i];
                t1 = __builtin_fmaf(dr[i], y[i], t1);
            }
            if (a.post) {
                meet.sum2(t0, t1);
                const float m0 = a.post_centred ? t0 * rD : 0.f, m1 = t1 * rD;
#pragma unroll
                for (int i = 0; i < 8; ++i) dr[i] = st.y * (dr[i] - m0 - y[i] * m1);
            }
            if (in) store8<DT, VEC>(a.dy, row, c, D, dr);
        }
        if (MANY && ends) {
            float sc[8], g[8];
            gate.get(g);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                all[i * MOST + tid] += g[i] * s0[i];
                all[(8 + i) * MOST + tid] += g[i] * s1[i];
            }
            param8(a.scale, c, D, 1.f, sc);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                g[i] = sc[i] * (qw[i] * s1[i] + qb[i] * s0[i]);
                s0[i] = s1[i] = 0.f;
            }
            if (in && a.dgate) store8<DT, VEC>(a.dgate, b, c, D, g);
            gate = ng;
            gate.get(g);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = sc[i] * g[i];
            end += a.L;
            ++b;
        }
    }
    if (MANY) {
#pragma unroll
        for (int i = 0; i < 8; ++i) { s0[i] = all[i * MOST + tid]; s1[i] = all[(8 + i) * MOST + tid]; }
    }
    float* p = a.part + (int64_t)blockIdx.x * 4 * D;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (c + i < D) { p[c + i] = s0[i]; p[D + c + i] = s1[i]; p[2 * D + c + i] = s2[i]; p[3 * D + c + i] = s3[i]; }
}

// sums over the chunks of a sample: part [B, chunks, 4, D] -> joint [B, 4, D], and the sample's dgate. COLS columns x 256 / COLS chunk lanes: 64 x 4, or
// 16 x 16 for long lists of chunks (4 samples of 768 chunks of 512: 75 us with 64 x 4).
// (`total` chunks in all: those of no sample in particular -- no gate, MANY -- stand in groups of JOIN, the last of which may be part full: in one
// group 1022 chunks of 1280 took 82 us)
constexpr int JOIN = 64;
template <int DT, int COLS>
__global__ __launch_bounds__(256) void norm_join_kernel(NormArgs a, float* joint, int total) {
    if constexpr (DT == 1) T16<true>::enter();
    constexpr int LANES = 256 / COLS;
    __shared__ float red[LANES][4][COLS];
    const int cl = threadIdx.x % COLS, kl = threadIdx.x / COLS, b = blockIdx.y, c = blockIdx.x * COLS + cl, D = a.D;
    float s[4] = {};
    if (c < D)
        for (int k = kl; k < min(a.chunks, total - b * a.chunks); k += LANES) {
            const float* p = a.part + ((int64_t)b * a.chunks + k) * 4 * D + c;
#pragma unroll
            for (int j = 0; j < 4; ++j) s[j] += p[j * D];
        }
#pragma unroll
    for (int j = 0; j < 4; ++j) red[kl][j][cl] = s[j];
    __syncthreads();
    if (c >= D || kl >= 4) return;
    const auto sum = [&](int j) {
        float t = red[0][j][cl];
#pragma unroll
        for (int k = 1; k < LANES; ++k) t += red[k][j][cl];
        return t;
    };
    if (joint != a.part) joint[((int64_t)b * 4 + kl) * D + c] = sum(kl);
    if (kl == 0 && a.dgate) {
        const float w = a.post_w ? a.post_w[c] : 1.f, q = a.post_b ? a.post_b[c] : 0.f;
        const float v = (a.scale ? a.scale[c] : 1.f) * (w * sum(1) + q * sum(0));
        if constexpr (DT == 0) static_cast<float*>(a.dgate)[(int64_t)b * D + c] = v;
        else static_cast<uint16_t*>(a.dgate)[(int64_t)b * D + c] = T16<DT == 1>::from_f32(v);
    }
}
// joint [B, 4, D] -> the parameters' gradients: 32 columns x 32 sample lanes
template <int DT>
__global__ __launch_bounds__(1024) void norm_params_kernel(NormArgs a, const float* joint) {
    __shared__ float red[32][5][32];
    const int cl = threadIdx.x & 31, bl = threadIdx.x >> 5, c = blockIdx.x * 32 + cl, D = a.D;
    float s[5] = {};                         // dscale, dw_post, dbias_post, dw_pre, dbias_pre
    if (c < D) {
        const float w = a.post_w ? a.post_w[c] : 1.f, q = a.post_b ? a.post_b[c] : 0.f, sc = a.scale ? a.scale[c] : 1.f;
        for (int b = bl; b < a.B; b += 32) {
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
    for (int k = 0; k < 32; ++k) t += red[k][bl][cl];
    float* out[5] = {a.d_scale, a.d_post_w, a.d_post_b, a.d_pre_w, a.d_pre_b};
    float* o = bl == 0 ? out[0] : bl == 1 ? out[1] : bl == 2 ? out[2] : bl == 3 ? out[3] : out[4];
    if (o) o[c] = t;
}

// Workgroups that walk the rows: what the 256 CUs hold at once (five waves per SIMD forward, three backward, as the registers allow), so
// that no second round is left over (rows of 1280: 2048 workgroups instead of 1536 took 98 us instead of 85)
int walkers(int threads, int waves_per_simd) { return 256 * std::max(1, 4 * waves_per_simd / (threads / 64)); }

bool vec_ok(const NormArgs& a) {
    uintptr_t m = 0;
    for (const void* p : {a.x, a.y, a.gate, a.dr, a.dz, (const void*)a.r, (const void*)a.z, (const void*)a.dx, (const void*)a.dy}) m |= (uintptr_t)p;
    return a.D % 8 == 0 && m % 16 == 0;
}
// Chunks of rows per sample; without a gate all rows are one sample. More short samples than workgroups: chunks of whole samples (the kernel's MANY),
// up to 16 rows to a sample, 2 where a row takes more than four waves (their registers do not hold MANY's sums beside a row's). us, forward and
// backward, a chunk per sample and MANY: samples x rows x D, bf16: 20000 x 1 x 256 528, 92; 9000 x 1 x 512 298, 107; 7000 x 16 x 512 481, 369; 7000 x
// 60 x 256 754, 922; 6000 x 1 x 4096 1049, 397; 600 x 2 x 4096 140, 130; 600 x 8 x 4096 254, 290; f32: 7000 x 4 x 512 321, 228; 600 x 8 x 4096 354, 447.
// One chunk per sample needs no copy for the sums over the samples (600 x 16 x 8192 bf16 872, 752 without).
bool plan(NormArgs& a) {
    if (!a.gate) { a.L *= a.B; a.B = 1; }
    const int wgs = walkers(64 * cdiv(a.D, 512), 3);
    const bool many = a.B > 2 * wgs && a.L <= (a.D <= 2048 ? 16 : 2);
    const int n = many ? a.B : a.L, want = many ? 4 * wgs : std::max(1, wgs / a.B);
    a.rows_per_chunk = cdiv(n, std::min(want, n));
    a.chunks = cdiv(n, a.rows_per_chunk);
    return many;
}
bool grouped(const NormArgs& a) { return !a.gate && a.chunks > JOIN; }
template <int DT>
int fwd(const NormArgs& a, hipStream_t st) {
    const int rows = a.B * a.L, threads = 64 * cdiv(a.D, 512);
    const unsigned grid = (unsigned)std::min(rows, walkers(threads, threads <= 256 ? 5 : 4));
    if (vec_ok(a)) {
        if (threads <= 256) norm_fwd_kernel<DT, true, 256><<<grid, threads, 0, st>>>(a, rows);
        else norm_fwd_kernel<DT, true, 1024><<<grid, threads, 0, st>>>(a, rows);
    } else {
        norm_fwd_kernel<DT, false, 1024><<<grid, threads, 0, st>>>(a, rows);
    }
    ISB_LAUNCHED("norm_fwd", st);
    return ISB_OK;
}
template <int DT, bool MANY>
void bwd_rows(const NormArgs& a, unsigned grid, hipStream_t st) {
    const int threads = 64 * cdiv(a.D, 512);
    if (vec_ok(a)) {
        if (threads <= 256) norm_bwd_kernel<DT, true, 256, MANY><<<grid, threads, 0, st>>>(a);
        else norm_bwd_kernel<DT, true, 1024, MANY><<<grid, threads, 0, st>>>(a);
    } else {
        norm_bwd_kernel<DT, false, 1024, MANY><<<grid, threads, 0, st>>>(a);
    }
}
template <int DT>
int bwd(NormArgs a, float* ws, hipStream_t st) {
    const bool many = plan(a);
    const int total = many ? a.chunks : a.B * a.chunks;
    a.part = ws;
    if (many) bwd_rows<DT, true>(a, (unsigned)total, st);
    else bwd_rows<DT, false>(a, (unsigned)total, st);
    if (many || grouped(a)) {                                // what is left to add up knows no gate
        a.B = cdiv(total, JOIN);
        a.chunks = JOIN;
        a.gate = nullptr;
        a.dgate = nullptr;
    }
    ISB_LAUNCHED("norm_bwd", st);
    float* joint = a.chunks == 1 ? ws : ws + (int64_t)total * 4 * a.D;
    if (joint != ws || a.dgate) {
        if (a.chunks > JOIN) norm_join_kernel<DT, 16><<<dim3(cdiv(a.D, 16), a.B), 256, 0, st>>>(a, joint, total);
        else norm_join_kernel<DT, 64><<<dim3(cdiv(a.D, 64), a.B), 256, 0, st>>>(a, joint, total);
        ISB_LAUNCHED("norm_join", st);
    }
    norm_params_kernel<DT><<<cdiv(a.D, 32), 1024, 0, st>>>(a, joint);
    ISB_LAUNCHED("norm_params", st);
    return ISB_OK;
}
}  // namespace

size_t norm_workspace(const NormArgs& a0) {
    NormArgs a = a0;
    if (plan(a) || grouped(a)) return ((size_t)a.chunks + cdiv(a.chunks, JOIN)) * 4 * a.D * sizeof(float);
    return ((size_t)a.B * a.chunks + (a.chunks == 1 ? 0 : a.B)) * 4 * a.D * sizeof(float);
}
int launch_norm_fwd(const NormArgs& a, int dtype, hipStream_t st) { return dtype == 0 ? fwd<0>(a, st) : dtype == 1 ? fwd<1>(a, st) : fwd<2>(a, st); }
int launch_norm_bwd(NormArgs a, int dtype, float* ws, hipStream_t st) { return dtype == 0 ? bwd<0>(a, ws, st) : dtype == 1 ? bwd<1>(a, ws, st) : bwd<2>(a, ws, st); }

}  // namespace isb
