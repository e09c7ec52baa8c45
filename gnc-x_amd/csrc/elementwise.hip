// elementwise.hip -- the small per-token kernels around the hot path, plus
// the block dequantiser used to prove the decoders bit-exact.
//   per-head RMSNorm      cpp:895-953    RMSNorm (fast path)  cpp:789-833
//   NEOX RoPE             cpp:1797-1862  SwiGLU               cpp:2038-2052
//   lm_head softcap       cpp:1726-1731  embedding row fetch  cpp:693-780
//   block decoders        cpp:85-112, 707-714, 734-759 and the dots' implicit
//                         Q4_0/Q4_K decoders (cpp:1023-1030, 1127-1178)
#include <hip/hip_runtime.h>

#include "gncx_act.h"
#include "gncx_device.h"
#include "gncx_launch.h"
#include "gncx_wave64.h"

namespace gncx {
namespace {

using namespace dev;

// One wave per head: the head is copied into LDS with coalesced loads, then
// head_inv_rms forms the reference's four sequential fp32 lane sums from the
// LDS copy (bit-exact with cpp:905-926) and the wave writes the result.  Heads
// longer than kHeadsMaxHd (whole-vector norms, n_heads = 1) read global memory.
constexpr int kHeadsMaxHd = 512;

__global__ __launch_bounds__(256) void rmsnorm_heads_kernel(float* __restrict v, const float* __restrict g,
                                                            int32_t n_heads, int32_t hd, float eps) {
#pragma clang fp contract(off)
    __shared__ float buf[4][kHeadsMaxHd];
    const int w = threadIdx.x >> 6;
    const int h = blockIdx.x * 4 + w;
    const int lane = threadIdx.x & 63;
    const bool active = h < n_heads;
    float* x = v + static_cast<size_t>(active ? h : 0) * hd;
    float* lx = buf[w];
    if (active)
        for (int i = lane; i < hd; i += 64) lx[i] = x[i];
    __syncthreads();
    if (!active) return;
    const float inv = head_inv_rms(lx, hd, eps, lane);
    for (int i = lane; i < hd; i += 64) {
        const float y = lx[i] * inv;
        x[i] = g ? y * g[i] : y;
    }
}

__global__ __launch_bounds__(256) void rmsnorm_heads_long_kernel(float* __restrict v, const float* __restrict g,
                                                                 int32_t n_heads, int32_t hd, float eps) {
#pragma clang fp contract(off)
    const int h = blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (h >= n_heads) return;
    float* x = v + static_cast<size_t>(h) * hd;
    const float inv = head_inv_rms(x, hd, eps, lane);
    for (int i = lane; i < hd; i += 64) {
        const float y = x[i] * inv;
        x[i] = g ? y * g[i] : y;
    }
}

// The 4-phase telemetry encode of one vector (reference cpp:842-889) by one
// work-group of kNormThreads: the largest |v| (at least 1e-9), the scale to
// the layer's integer range 9 R_k (R_k the repunit of k ones), then per
// element the rounded integer, its diagonal digit d (nearest multiple of R_k,
// at most 9), the residual from d R_k and the two sign bits, packed as the
// 4-byte token {phase, d, |residual| mod 2^16}.  Every float step is the
// reference's, correctly rounded and uncontracted, so the tokens are
// bit-exact.  qscale[0] receives the quant scale and qscale[1] (as a
// uint32) the cancellation count sum_d min(#positive, #negative) over the
// digits d (cpp:882-887).  red: kNormThreads / 64 floats of LDS.
// One element of the encode: the token, and the counter of its (sign, digit)
// pair (0-9: val >= 0, 10-19: val < 0) for the cancellation count.
struct EncScale {
    int64_t r_k;
    float to_int, inv_rk, half_rk;
};
template <class I>
__device__ __forceinline__ uint32_t encode_value(float v, const EncScale& e, uint32_t& ctr) {
#pragma clang fp contract(off)
    const I val = static_cast<I>(rintf(__fmul_rn(v, e.to_int)));
    const I av = val >= 0 ? val : -val;
    int32_t d = static_cast<int32_t>(__fmul_rn(__fadd_rn(static_cast<float>(av), e.half_rk), e.inv_rk));
    if (d > 9) d = 9;
    const I anchor = static_cast<I>(d) * static_cast<I>(e.r_k);
    const I res = val - (val >= 0 ? anchor : -anchor);
    const uint32_t ares = static_cast<uint32_t>(static_cast<uint16_t>(res >= 0 ? res : -res));
    const uint32_t phase = (val >= 0 ? 2u : 0u) | (res >= 0 ? 1u : 0u);
    ctr = static_cast<uint32_t>(d) + (val >= 0 ? 0u : 10u);
    return phase | (static_cast<uint32_t>(d) << 8) | (ares << 16);
}
// Up to k = 8 every integer of the encode (|val| <= 9 R_k < 10^9, the residual
// below 2 x 10^9) fits 32 bits, and the 32-bit steps give the 64-bit results.
constexpr int32_t kEnc32MaxK = 8;

// the scale of the layer's range from the largest |v| m (qscale[0] = m / 9 R_k)
__device__ __forceinline__ EncScale encode_scale(float m, int32_t lay_k, float* __restrict qscale) {
#pragma clang fp contract(off)
    EncScale e;
    e.r_k = 1;
    for (int i = 0; i < lay_k; ++i) e.r_k = e.r_k * 10 + 1;
    const float target = static_cast<float>(9 * e.r_k);
    e.to_int = __fdiv_rn(target, m);
    if (threadIdx.x == 0) *qscale = __fdiv_rn(m, target);
    e.inv_rk = __fdiv_rn(1.0f, static_cast<float>(e.r_k));
    e.half_rk = static_cast<float>(e.r_k >> 1);
    return e;
}

__device__ void encode_row(const float* v, int32_t dim, int32_t lay_k, uint32_t* __restrict tokens,
                           float* __restrict qscale, float* red) {
    __shared__ uint32_t signs[20];
    if (threadIdx.x < 20) signs[threadIdx.x] = 0;
    float m = 1e-9f;
    for (int32_t i = threadIdx.x; i < dim; i += blockDim.x) {
        const float a = fabsf(v[i]);
        m = a > m ? a : m;
    }
    m = wave_max(m);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    m = red[0];
    for (int w = 1; w < static_cast<int>(blockDim.x / 64); ++w) m = red[w] > m ? red[w] : m;
    const EncScale e = encode_scale(m, lay_k, qscale);
    for (int32_t i = threadIdx.x; i < dim; i += blockDim.x) {
        uint32_t ctr;
        tokens[i] = lay_k <= kEnc32MaxK ? encode_value<int32_t>(v[i], e, ctr) : encode_value<int64_t>(v[i], e, ctr);
        __hip_atomic_fetch_add(&signs[ctr], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        uint32_t c = 0;
        for (int d = 0; d < 10; ++d) c += signs[d] < signs[10 + d] ? signs[d] : signs[10 + d];
        reinterpret_cast<uint32_t*>(qscale)[1] = c;
    }
}

// RMSNorm of one row per work-group (cpp:789-833): x and gamma are read once
// as float4 (kept in registers for rows up to 16384 values), the sum of
// squares is a fp32 tree over the work-group, y = (x * inv) * gamma.
constexpr int kNormThreads = 1024;
constexpr int kNormRegs = 4;  // float4 per thread held in registers

// The encode of a row whose normalised values a work-group of kNormThreads
// holds in registers (y[j]: float4 t = threadIdx.x + kNormThreads j, t < n4):
// no second pass over memory, tokens stored as uint4 (16-byte aligned), and
// the (sign, digit) counts formed per wave with ballots instead of LDS
// atomics on 20 addresses.  Max, tokens and counts are those of encode_row
// (a max and integer counts do not depend on the order).
__device__ void encode_regs(const float4 (&y)[kNormRegs], int32_t n4, int32_t lay_k, uint32_t* __restrict tokens,
                            float* __restrict qscale) {
    __shared__ float red[kNormThreads / 64];
    __shared__ uint32_t cnt[kNormThreads / 64][20];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    float m = 1e-9f;
#pragma unroll
    for (int j = 0; j < kNormRegs; ++j) {
        if (tid + kNormThreads * j < n4) {
            const float a0 = fabsf(y[j].x), a1 = fabsf(y[j].y), a2 = fabsf(y[j].z), a3 = fabsf(y[j].w);
            m = a0 > m ? a0 : m;
            m = a1 > m ? a1 : m;
            m = a2 > m ? a2 : m;
            m = a3 > m ? a3 : m;
        }
    }
    m = wave_max(m);
    if (lane == 0) red[w] = m;
    __syncthreads();
    m = red[0];
#pragma unroll
    for (int i = 1; i < kNormThreads / 64; ++i) m = red[i] > m ? red[i] : m;
    const EncScale e = encode_scale(m, lay_k, qscale);
    uint4* t4 = reinterpret_cast<uint4*>(tokens);
    const bool small = lay_k <= kEnc32MaxK;
    uint32_t n[20] = {};
#pragma unroll
    for (int j = 0; j < kNormRegs; ++j) {
        if (kNormThreads * j >= n4) break;  // no thread holds float4 j
        const int32_t t = tid + kNormThreads * j;
        uint32_t ctr[4] = {20u, 20u, 20u, 20u};  // 20: counted nowhere
        if (t < n4) {
            uint4 tk;
            const float* yj = &y[j].x;
#pragma unroll
            for (int q = 0; q < 4; ++q)
                (&tk.x)[q] = small ? encode_value<int32_t>(yj[q], e, ctr[q]) : encode_value<int64_t>(yj[q], e, ctr[q]);
            t4[t] = tk;
        }
#pragma unroll
        for (uint32_t c = 0; c < 20; ++c)
#pragma unroll
            for (int q = 0; q < 4; ++q) n[c] += static_cast<uint32_t>(__popcll(__ballot(ctr[q] == c)));
    }
    if (lane == 0)
#pragma unroll
        for (int c = 0; c < 20; ++c) cnt[w][c] = n[c];
    __syncthreads();
    if (w == 0) {
        // lane d < 10 sums digit d's two counts over the waves; the ten
        // minima meet in one wave sum (integers below 2^24: exact in fp32)
        float mn = 0.0f;
        if (lane < 10) {
            uint32_t pos = 0, neg = 0;
#pragma unroll
            for (int i = 0; i < kNormThreads / 64; ++i) {
                pos += cnt[i][lane];
                neg += cnt[i][10 + lane];
            }
            mn = static_cast<float>(pos < neg ? pos : neg);
        }
        mn = wave_sum(mn);
        if (lane == 0) reinterpret_cast<uint32_t*>(qscale)[1] = static_cast<uint32_t>(mn);
    }
}

// ADD: x is the residual stream h (row blockIdx.x), updated in place to h + r
// before it is normalised -- the fp32 add of the separate vec_add kernel, so
// the result is the same bit for bit.  ENC: the 4-phase encode of the
// normalised row follows in the same work-group (one row).
template <bool ADD, bool ENC = false>
// (x and xo are the same row under ADD: no __restrict on the row pointers)
__global__ __launch_bounds__(kNormThreads) void rmsnorm_kernel(const float* x, const float* __restrict g,
                                                               int32_t dim, float eps, float* out, int32_t vec4,
                                                               const float* r, float* xo, int32_t lay_k = 0,
                                                               uint32_t* tokens = nullptr, float* qscale = nullptr) {
#pragma clang fp contract(off)
    __shared__ float part[kNormThreads / 64];
    const float* xr = x + static_cast<size_t>(blockIdx.x) * dim;
    float* yr = out + static_cast<size_t>(blockIdx.x) * dim;
    if (ADD) {  // one row per work-group: its residual row and delta row
        r += static_cast<size_t>(blockIdx.x) * dim;
        xo += static_cast<size_t>(blockIdx.x) * dim;
    }
    const int tid = threadIdx.x;
    float s = 0.0f;
    float4 xv[kNormRegs], gv[kNormRegs];
    const int32_t n4 = vec4 ? dim / 4 : 0;
    const float4* x4 = reinterpret_cast<const float4*>(xr);
    const float4* g4 = reinterpret_cast<const float4*>(g);
    const float4* r4 = reinterpret_cast<const float4*>(r);
    float4* xo4 = reinterpret_cast<float4*>(xo);
    auto add4 = [](float4 a, float4 b) { return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); };
#pragma unroll
    for (int j = 0; j < kNormRegs; ++j) {
        const int32_t t = tid + kNormThreads * j;
        if (t < n4) {
            xv[j] = x4[t];
            if (ADD) {
                xv[j] = add4(xv[j], r4[t]);
                xo4[t] = xv[j];
            }
            gv[j] = g4[t];
            s += xv[j].x * xv[j].x + xv[j].y * xv[j].y + xv[j].z * xv[j].z + xv[j].w * xv[j].w;
        }
    }
    for (int32_t t = tid + kNormThreads * kNormRegs; t < n4; t += kNormThreads) {
        float4 a = x4[t];
        if (ADD) {
            a = add4(a, r4[t]);
            xo4[t] = a;
        }
        s += a.x * a.x + a.y * a.y + a.z * a.z + a.w * a.w;
    }
    for (int32_t i = 4 * n4 + tid; i < dim; i += kNormThreads) {
        float a = xr[i];
        if (ADD) {
            a = a + r[i];
            xo[i] = a;
        }
        s += a * a;
    }
    // rows past the registers are read again below: from xo, which now holds h + r
    if (ADD) {
        xr = xo;
        x4 = reinterpret_cast<const float4*>(xo);
    }
    s = wave_sum(s);
    if ((tid & 63) == 0) part[tid >> 6] = s;
    __syncthreads();
    float tot = 0.0f;
#pragma unroll
    for (int w = 0; w < kNormThreads / 64; ++w) tot += part[w];
    const float inv = 1.0f / sqrtf(tot / static_cast<float>(dim) + eps);
    float4* y4 = reinterpret_cast<float4*>(yr);
    float4 yv[kNormRegs];
#pragma unroll
    for (int j = 0; j < kNormRegs; ++j) {
        const int32_t t = tid + kNormThreads * j;
        yv[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (t < n4) {
            yv[j] = make_float4(xv[j].x * inv * gv[j].x, xv[j].y * inv * gv[j].y, xv[j].z * inv * gv[j].z,
                                xv[j].w * inv * gv[j].w);
            y4[t] = yv[j];
        }
    }
    for (int32_t t = tid + kNormThreads * kNormRegs; t < n4; t += kNormThreads) {
        const float4 a = x4[t], b = g4[t];
        y4[t] = make_float4(a.x * inv * b.x, a.y * inv * b.y, a.z * inv * b.z, a.w * inv * b.w);
    }
    for (int32_t i = 4 * n4 + tid; i < dim; i += kNormThreads) yr[i] = xr[i] * inv * g[i];
    if constexpr (ENC) {
        // the whole row in registers and 16-byte token stores: encode from
        // the registers; otherwise from the row just stored
        if (4 * n4 == dim && n4 <= kNormThreads * kNormRegs && (reinterpret_cast<uintptr_t>(tokens) & 15u) == 0) {
            encode_regs(yv, n4, lay_k, tokens, qscale);
            return;
        }
        __threadfence_block();
        __syncthreads();
        encode_row(yr, dim, lay_k, tokens, qscale, part);
    }
}

__global__ void rope_kernel(float* __restrict q, float* __restrict k, RopeTable t, int32_t n_heads,
                            int32_t n_kv, int32_t hd) {
#pragma clang fp contract(off)
    const int half = hd / 2;
    const int total = (n_heads + n_kv) * half;
    for (int idx = blockIdx.x * blockDim.x + threadIdx.x; idx < total; idx += gridDim.x * blockDim.x) {
        const int h = idx / half, i = idx % half;
        float* v = h < n_heads ? (q ? q + static_cast<size_t>(h) * hd : nullptr)
                               : (k ? k + static_cast<size_t>(h - n_heads) * hd : nullptr);
        if (!v) continue;
        const float x1 = v[i], x2 = v[i + half];
        v[i] = x1 * t.c[i] - x2 * t.s[i];
        v[i + half] = x2 * t.c[i] + x1 * t.s[i];
    }
}

__global__ void swiglu_kernel(const float* __restrict g, const float* __restrict u, int32_t n,
                              float* __restrict out) {
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < n; i += gridDim.x * blockDim.x)
        out[i] = swiglu_value(g[i], u[i]);
}

// tanh-approximated GELU of the gate times up, in the reference's order of
// operations (cpp:2024-2030) with no contraction into fused multiply-adds.
__global__ void geglu_kernel(const float* __restrict g, const float* __restrict u, int32_t n,
                             float* __restrict out) {
    constexpr float kSqrt2OverPi = 0.7978845608028654f;
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < n; i += gridDim.x * blockDim.x) {
        const float x = g[i];
        const float cube = __fmul_rn(__fmul_rn(__fmul_rn(0.044715f, x), x), x);
        const float t = tanhf(__fmul_rn(kSqrt2OverPi, __fadd_rn(x, cube)));
        out[i] = __fmul_rn(__fmul_rn(__fmul_rn(0.5f, x), __fadd_rn(1.0f, t)), u[i]);
    }
}

__global__ void vec_add_kernel(float* __restrict y, const float* __restrict x, int32_t n) {
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < n; i += gridDim.x * blockDim.x) y[i] += x[i];
}

__global__ void softcap_kernel(float* __restrict y, int32_t n, float cap) {
    const float inv = __fdiv_rn(1.0f, cap);
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < n; i += gridDim.x * blockDim.x)
        y[i] = __fmul_rn(tanhf(__fmul_rn(y[i], inv)), cap);
}

// Decode element e of a row (all decoders are exact: every product below is
// representable in fp32, except where the reference also rounds).
__device__ __forceinline__ float decode_elem(int32_t type, const uint8_t* __restrict row, int32_t e, float scale) {
    if (type == kQ4_0) {
        const uint8_t* blk = row + static_cast<size_t>(e / 32) * 18;
        const int j = e % 32;
        const float d = half_bits_to_float(ld_u16(blk));
        const int b = blk[2 + (j & 15)];
        const int qv = (j < 16 ? (b & 15) : (b >> 4)) - 8;
        return __fmul_rn(d, static_cast<float>(qv));
    }
    if (type == kQ8_0) {
        const uint8_t* blk = row + static_cast<size_t>(e / 32) * 34;
        const float d = __fmul_rn(half_bits_to_float(ld_u16(blk)), scale);
        return __fmul_rn(static_cast<float>(static_cast<int8_t>(blk[2 + e % 32])), d);
    }
    if (type == kQ4_K) {
        const uint8_t* blk = row + static_cast<size_t>(e / 256) * 144;
        const int r = e % 256, c = r / 64, hi = (r % 64) / 32, l = r % 32;
        const uint32_t s0 = blk[4] | (blk[5] << 8) | (blk[6] << 16) | (static_cast<uint32_t>(blk[7]) << 24);
        const uint32_t s1 = blk[8] | (blk[9] << 8) | (blk[10] << 16) | (static_cast<uint32_t>(blk[11]) << 24);
        const uint32_t s2 = blk[12] | (blk[13] << 8) | (blk[14] << 16) | (static_cast<uint32_t>(blk[15]) << 24);
        int sc, mn;
        k4_scale_min(2 * c + hi, s0, s1, s2, sc, mn);
        const float d = half_bits_to_float(ld_u16(blk)), dmin = half_bits_to_float(ld_u16(blk + 2));
        const int b = blk[16 + 32 * c + l];
        const int qv = hi ? (b >> 4) : (b & 15);
        return __fsub_rn(__fmul_rn(__fmul_rn(d, static_cast<float>(sc)), static_cast<float>(qv)),
                         __fmul_rn(dmin, static_cast<float>(mn)));
    }
    if (type == kQ6_K) {
        const uint8_t* blk = row + static_cast<size_t>(e / 256) * 210;
        const int r = e % 256, h = r / 128, rr = r % 128, grp = rr / 32, l = rr % 32;
        const uint8_t* ql = blk + 64 * h;
        const uint8_t* qh = blk + 128 + 32 * h;
        const int8_t* sc = reinterpret_cast<const int8_t*>(blk + 192 + 8 * h);
        const int lo4 = (grp & 1) ? ql[l + 32] : ql[l];
        const int low = (grp >= 2) ? (lo4 >> 4) : (lo4 & 15);
        const int qv = (low | (((qh[l] >> (2 * grp)) & 3) << 4)) - 32;
        const float d = __fmul_rn(half_bits_to_float(ld_u16(blk + 208)), scale);
        return __fmul_rn(__fmul_rn(d, static_cast<float>(sc[l / 16 + 2 * grp])), static_cast<float>(qv));
    }
    // BF16
    return __fmul_rn(__uint_as_float(ld_u16(row + static_cast<size_t>(e) * 2) << 16), scale);
}

__global__ void dequant_kernel(int32_t type, const uint8_t* __restrict w, size_t rb, int32_t k, int32_t n,
                               float* __restrict out) {
    const size_t total = static_cast<size_t>(k) * n;
    for (size_t i = static_cast<size_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
         i += static_cast<size_t>(gridDim.x) * blockDim.x) {
        const int32_t r = static_cast<int32_t>(i / k), e = static_cast<int32_t>(i % k);
        out[i] = decode_elem(type, w + static_cast<size_t>(r) * rb, e, 1.0f);
    }
}

__global__ void fetch_embedding_kernel(int32_t type, const uint8_t* __restrict row, int32_t dim, float scale,
                                       float* __restrict out) {
    for (int e = blockIdx.x * blockDim.x + threadIdx.x; e < dim; e += gridDim.x * blockDim.x)
        out[e] = decode_elem(type, row, e, scale);
}

// The row of a token read from device memory (a decode loop that feeds its
// own argmax back without a host round trip).  Rows of tokens outside
// [0, vocab) are not read: the output is left as it is.
__global__ void fetch_embedding_dev_kernel(int32_t type, const uint8_t* __restrict table, const int32_t* token,
                                           int32_t vocab, size_t rbytes, int32_t dim, float scale,
                                           float* __restrict out) {
    const int32_t t = *token;
    if (t < 0 || t >= vocab) return;
    const uint8_t* row = table + static_cast<size_t>(t) * rbytes;
    for (int e = blockIdx.x * blockDim.x + threadIdx.x; e < dim; e += gridDim.x * blockDim.x)
        out[e] = decode_elem(type, row, e, scale);
}

// Rows of `count` tokens (ids already checked against the table's rows), one
// y-block of the grid per token.
__global__ void fetch_embedding_rows_kernel(int32_t type, const uint8_t* __restrict table, const int32_t* tokens,
                                            size_t rbytes, int32_t dim, float scale, float* __restrict out) {
    const uint8_t* row = table + static_cast<size_t>(tokens[blockIdx.y]) * rbytes;
    float* o = out + static_cast<size_t>(blockIdx.y) * dim;
    for (int e = blockIdx.x * blockDim.x + threadIdx.x; e < dim; e += gridDim.x * blockDim.x)
        o[e] = decode_elem(type, row, e, scale);
}

// Index of the largest value (the first one among equal maxima; NaN never
// wins), as torch.argmax and the greedy pick of the streamer's sampler take
// it.  Two launches: argmax_part_kernel reduces contiguous chunks of
// kArgmaxChunk values (coalesced float4 loads, several in flight per thread)
// to (value, index) pairs, argmax_final_kernel reduces the pairs.
constexpr int kArgmaxThreads = 256;
constexpr int kArgmaxChunk = 4096;
constexpr int kArgmaxMaxParts = 1024;

struct ArgBest {
    float v;
    int32_t i;  // INT32_MAX: no candidate
};
__device__ __forceinline__ ArgBest arg_better(ArgBest a, ArgBest b) {
    // b replaces a when it is larger, or equal with a smaller index; NaN never wins
    const bool take = b.i != INT32_MAX && (a.i == INT32_MAX || b.v > a.v || (b.v == a.v && b.i < a.i));
    return take ? b : a;
}
__device__ ArgBest block_argmax(ArgBest b) {
    __shared__ float sv[kArgmaxThreads];
    __shared__ int32_t si[kArgmaxThreads];
    sv[threadIdx.x] = b.v;
    si[threadIdx.x] = b.i;
    __syncthreads();
    for (int h = kArgmaxThreads / 2; h > 0; h >>= 1) {
        if (static_cast<int>(threadIdx.x) < h) {
            const ArgBest r = arg_better({sv[threadIdx.x], si[threadIdx.x]}, {sv[threadIdx.x + h], si[threadIdx.x + h]});
            sv[threadIdx.x] = r.v;
            si[threadIdx.x] = r.i;
        }
        __syncthreads();
    }
    return {sv[0], si[0]};
}

__global__ __launch_bounds__(kArgmaxThreads) void argmax_part_kernel(const float* __restrict x, int32_t n,
                                                                     float* __restrict pv, int32_t* __restrict pi) {
    const int32_t base = blockIdx.x * kArgmaxChunk;
    const int32_t end = min(n, base + kArgmaxChunk);
    ArgBest b{-INFINITY, INT32_MAX};
    // 4 values per thread per step, 4 steps: the whole chunk in flight at once
    float vals[kArgmaxChunk / kArgmaxThreads];
#pragma unroll
    for (int s = 0; s < kArgmaxChunk / (4 * kArgmaxThreads); ++s) {
        const int32_t i = base + 4 * (s * kArgmaxThreads + static_cast<int32_t>(threadIdx.x));
        if (i + 3 < end && (n & 3) == 0) {
            const float4 v = *reinterpret_cast<const float4*>(x + i);
            vals[4 * s] = v.x;
            vals[4 * s + 1] = v.y;
            vals[4 * s + 2] = v.z;
            vals[4 * s + 3] = v.w;
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) vals[4 * s + c] = i + c < end ? x[i + c] : NAN;
        }
    }
#pragma unroll
    for (int s = 0; s < kArgmaxChunk / (4 * kArgmaxThreads); ++s)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int32_t i = base + 4 * (s * kArgmaxThreads + static_cast<int32_t>(threadIdx.x)) + c;
            const float v = vals[4 * s + c];
            if (v == v) b = arg_better(b, {v, i});
        }
    b = block_argmax(b);
    if (threadIdx.x == 0) {
        pv[blockIdx.x] = b.v;
        pi[blockIdx.x] = b.i;
    }
}

__global__ __launch_bounds__(kArgmaxThreads) void argmax_final_kernel(const float* __restrict pv,
                                                                      const int32_t* __restrict pi, int32_t parts,
                                                                      int32_t* __restrict out, int32_t* __restrict log) {
    ArgBest b{-INFINITY, INT32_MAX};
    for (int32_t p = threadIdx.x; p < parts; p += kArgmaxThreads) b = arg_better(b, {pv[p], pi[p]});
    b = block_argmax(b);
    if (threadIdx.x == 0) {
        const int32_t r = b.i == INT32_MAX ? 0 : b.i;
        *out = r;
        if (log) *log = r;
    }
}

int grid_for(size_t n, int threads) {
    size_t g = (n + threads - 1) / threads;
    if (g > 4096) g = 4096;
    return g < 1 ? 1 : static_cast<int>(g);
}

}  // namespace

hipError_t launch_rmsnorm_heads(float* v, const float* gamma, int32_t n_heads, int32_t head_dim, float eps,
                                hipStream_t stream) {
    if (n_heads <= 0 || head_dim <= 0) return hipSuccess;
    if (head_dim <= kHeadsMaxHd)
        hipLaunchKernelGGL(rmsnorm_heads_kernel, dim3((n_heads + 3) / 4), dim3(256), 0, stream, v, gamma, n_heads,
                           head_dim, eps);
    else
        hipLaunchKernelGGL(rmsnorm_heads_long_kernel, dim3((n_heads + 3) / 4), dim3(256), 0, stream, v, gamma,
                           n_heads, head_dim, eps);
    return hipGetLastError();
}

hipError_t launch_rmsnorm(const float* x, const float* gamma, int32_t rows, int32_t dim, float eps, float* out,
                          hipStream_t stream) {
    if (rows <= 0 || dim <= 0) return hipSuccess;
    const uintptr_t al = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(gamma) |
                         reinterpret_cast<uintptr_t>(out);
    const int32_t vec4 = (dim % 4 == 0 && (al & 15u) == 0) ? 1 : 0;
    hipLaunchKernelGGL(rmsnorm_kernel<false>, dim3(rows), dim3(kNormThreads), 0, stream, x, gamma, dim, eps, out,
                       vec4, nullptr, nullptr);
    return hipGetLastError();
}

hipError_t launch_add_rmsnorm_rows(float* h, const float* r, const float* gamma, int32_t rows, int32_t dim, float eps,
                                   float* out, hipStream_t stream) {
    if (rows <= 0 || dim <= 0) return hipSuccess;
    const uintptr_t al = reinterpret_cast<uintptr_t>(h) | reinterpret_cast<uintptr_t>(r) |
                         reinterpret_cast<uintptr_t>(gamma) | reinterpret_cast<uintptr_t>(out);
    const int32_t vec4 = (dim % 4 == 0 && (al & 15u) == 0) ? 1 : 0;
    hipLaunchKernelGGL(rmsnorm_kernel<true>, dim3(rows), dim3(kNormThreads), 0, stream, h, gamma, dim, eps, out, vec4,
                       r, h);
    return hipGetLastError();
}

hipError_t launch_add_rmsnorm(float* h, const float* r, const float* gamma, int32_t dim, float eps, float* out,
                              hipStream_t stream) {
    if (dim <= 0) return hipSuccess;
    const uintptr_t al = reinterpret_cast<uintptr_t>(h) | reinterpret_cast<uintptr_t>(r) |
                         reinterpret_cast<uintptr_t>(gamma) | reinterpret_cast<uintptr_t>(out);
    const int32_t vec4 = (dim % 4 == 0 && (al & 15u) == 0) ? 1 : 0;
    hipLaunchKernelGGL(rmsnorm_kernel<true>, dim3(1), dim3(kNormThreads), 0, stream, h, gamma, dim, eps, out, vec4, r,
                       h);
    return hipGetLastError();
}

hipError_t launch_rope(float* q, float* k, const RopeTable& table, int32_t n_heads, int32_t n_kv_heads,
                       int32_t head_dim, hipStream_t stream) {
    if (head_dim / 2 > kMaxRopeHalf || table.half * 2 != head_dim) return hipErrorInvalidValue;
    const size_t work = static_cast<size_t>(n_heads + n_kv_heads) * (head_dim / 2);
    if (work == 0) return hipSuccess;
    hipLaunchKernelGGL(rope_kernel, dim3(grid_for(work, 256)), dim3(256), 0, stream, q, k, table, n_heads,
                       n_kv_heads, head_dim);
    return hipGetLastError();
}

hipError_t launch_vec_add(float* y, const float* x, int32_t n, hipStream_t stream) {
    if (n <= 0) return hipSuccess;
    hipLaunchKernelGGL(vec_add_kernel, dim3(grid_for(n, 256)), dim3(256), 0, stream, y, x, n);
    return hipGetLastError();
}

hipError_t launch_swiglu(const float* gate, const float* up, int32_t n, float* out, hipStream_t stream) {
    if (n <= 0) return hipSuccess;
    hipLaunchKernelGGL(swiglu_kernel, dim3(grid_for(n, 256)), dim3(256), 0, stream, gate, up, n, out);
    return hipGetLastError();
}

hipError_t launch_geglu(const float* gate, const float* up, int32_t n, float* out, hipStream_t stream) {
    if (n <= 0) return hipSuccess;
    hipLaunchKernelGGL(geglu_kernel, dim3(grid_for(n, 256)), dim3(256), 0, stream, gate, up, n, out);
    return hipGetLastError();
}

hipError_t launch_rmsnorm_encode(const float* x, const float* gamma, int32_t dim, float eps, float* out,
                                 int32_t layer_k, uint32_t* tokens, float* qscale, hipStream_t stream) {
    if (dim <= 0) return hipSuccess;
    const uintptr_t al = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(gamma) |
                         reinterpret_cast<uintptr_t>(out);
    const int32_t vec4 = (dim % 4 == 0 && (al & 15u) == 0) ? 1 : 0;
    const int32_t k = layer_k < 0 ? 0 : (layer_k > 17 ? 17 : layer_k);
    hipLaunchKernelGGL((rmsnorm_kernel<false, true>), dim3(1), dim3(kNormThreads), 0, stream, x, gamma, dim, eps, out,
                       vec4, nullptr, nullptr, k, tokens, qscale);
    return hipGetLastError();
}

hipError_t launch_softcap(float* y, int32_t n, float softcap, hipStream_t stream) {
    if (n <= 0 || !(softcap > 0.0f)) return hipSuccess;
    hipLaunchKernelGGL(softcap_kernel, dim3(grid_for(n, 256)), dim3(256), 0, stream, y, n, softcap);
    return hipGetLastError();
}

hipError_t launch_dequant(int32_t type, const uint8_t* w, int32_t k, int32_t n, float* out, hipStream_t stream) {
    if (!type_supported(type)) return hipErrorInvalidValue;
    if (k <= 0 || n <= 0) return hipSuccess;
    if (k % block_elems(type) != 0 || (reinterpret_cast<uintptr_t>(w) & 1u)) return hipErrorInvalidValue;
    const size_t total = static_cast<size_t>(k) * n;
    hipLaunchKernelGGL(dequant_kernel, dim3(grid_for(total, 256)), dim3(256), 0, stream, type, w,
                       row_bytes(type, k), k, n, out);
    return hipGetLastError();
}

hipError_t launch_fetch_embedding(int32_t type, const uint8_t* table, int32_t token, int32_t dim, float scale,
                                  float* out, hipStream_t stream) {
    if (type != kQ8_0 && type != kQ6_K && type != kBF16) return hipErrorInvalidValue;
    if (dim <= 0) return hipSuccess;
    const uint8_t* row = table + static_cast<size_t>(token) * row_bytes(type, dim);
    hipLaunchKernelGGL(fetch_embedding_kernel, dim3(grid_for(dim, 256)), dim3(256), 0, stream, type, row, dim,
                       scale, out);
    return hipGetLastError();
}

hipError_t launch_fetch_embedding_rows(int32_t type, const uint8_t* table, const int32_t* tokens, int32_t count,
                                       int32_t dim, float scale, float* out, hipStream_t stream) {
    if (type != kQ8_0 && type != kQ6_K && type != kBF16) return hipErrorInvalidValue;
    if (dim <= 0 || count <= 0) return hipSuccess;
    if (count > 65535) return hipErrorInvalidValue;
    hipLaunchKernelGGL(fetch_embedding_rows_kernel, dim3(grid_for(dim, 256), count), dim3(256), 0, stream, type,
                       table, tokens, row_bytes(type, dim), dim, scale, out);
    return hipGetLastError();
}

hipError_t launch_fetch_embedding_dev(int32_t type, const uint8_t* table, const int32_t* token, int32_t vocab,
                                      int32_t dim, float scale, float* out, hipStream_t stream) {
    if (dim <= 0 || vocab <= 0) return hipSuccess;
    hipLaunchKernelGGL(fetch_embedding_dev_kernel, dim3(grid_for(dim, 256)), dim3(256), 0, stream, type, table, token,
                       vocab, row_bytes(type, dim), dim, scale, out);
    return hipGetLastError();
}

size_t argmax_workspace_bytes(int32_t n) {
    const size_t parts = n > 0 ? (static_cast<size_t>(n) + kArgmaxChunk - 1) / kArgmaxChunk : 0;
    return parts * (sizeof(float) + sizeof(int32_t));
}

hipError_t launch_argmax(const float* x, int32_t n, int32_t* out, int32_t* log, void* workspace, size_t ws_bytes,
                         hipStream_t stream) {
    if (n <= 0 || (reinterpret_cast<uintptr_t>(x) & 15u) != 0) return hipErrorInvalidValue;
    const int32_t parts = (n + kArgmaxChunk - 1) / kArgmaxChunk;
    if (parts > kArgmaxMaxParts || ws_bytes < argmax_workspace_bytes(n)) return hipErrorInvalidValue;
    float* pv = static_cast<float*>(workspace);
    int32_t* pi = reinterpret_cast<int32_t*>(pv + parts);
    hipLaunchKernelGGL(argmax_part_kernel, dim3(parts), dim3(kArgmaxThreads), 0, stream, x, n, pv, pi);
    hipLaunchKernelGGL(argmax_final_kernel, dim3(1), dim3(kArgmaxThreads), 0, stream, pv, pi, parts, out, log);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Choosing between continuations of one sequence and rearranging the KV caches
// after the choice: the rows of an accepted draft path, beam search's
// selection over beams and vocabulary, and the reordering of the beams' caches.
namespace {

constexpr int kCandThreads = 256;
constexpr int kLayerGroup = 64;  // layers of a launch: their cache addresses travel in the kernel arguments

struct LayerCaches {
    float* c[2 * kLayerGroup];  // layer l: its k cache at 2 l, its v cache at 2 l + 1
};

// ---- rows of an accepted path ----------------------------------------------
// Row row0 + i of every cache becomes the old row row0 + rows[i], rows
// ascending.  A thread owns one column (W floats) of one cache and moves its rows
// in order, kAtOnce loads before their stores: as rows[i] >= i and the rows
// ascend, no row is overwritten before it is read, and no thread touches
// another's column, so the move is in place without a barrier.  Rows that stay
// (rows[i] == i, the first ones only) are left out by the caller.
// Bound by memory, a round of loads and stores after the other: 400 of 512 rows of
// 1024 in 72 caches (118 MB read and written) 72 us with 16 at once, 50 (4.7 TB/s)
// with 64; 4 of 16 rows 4.2.  The rows are read as one vector, a round ahead: each
// of sixteen scalar loads from the arguments, in host memory, was waited for.
struct KeepParams {
    LayerCaches caches;
    int32_t kv_dim, n;
    size_t row0;
    uint16_t rows[kMaxKeepRows];  // 0 past n
};

template <int W, int kAtOnce>
__global__ __launch_bounds__(64) void keep_rows_kernel(KeepParams p) {
    typedef float vec __attribute__((ext_vector_type(W)));
    const int lane = threadIdx.x, d = W * static_cast<int>(blockIdx.x * 64 + lane);
    const bool in = d < p.kv_dim;
    float* c = p.caches.c[blockIdx.y] + p.row0 * p.kv_dim + (in ? d : 0);
    // lane u: where row i + u comes from (past the end row 0, read for nothing)
    int next = p.rows[lane % kAtOnce];
    for (int i = 0; i < p.n; i += kAtOnce) {
        const int from = next;
        next = p.rows[min(i + kAtOnce + lane % kAtOnce, kMaxKeepRows - 1)];
        vec v[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u)
            v[u] = *reinterpret_cast<const vec*>(c + static_cast<size_t>(__builtin_amdgcn_readlane(from, u)) * p.kv_dim);
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u)
            if (in && i + u < p.n) *reinterpret_cast<vec*>(c + static_cast<size_t>(i + u) * p.kv_dim) = v[u];
    }
}

// ---- reordering of beams ------------------------------------------------------
// Rows [row0, row0 + n_rows) of beam b become those of beam parents[b].  A
// thread owns U float4 of a cache's rows in all beams: it loads every moving
// beam's new values before it stores any, so the exchange is in place with no
// second copy of the caches.  A parent outside [0, n_beams) leaves its beam as it
// is.  Bound by memory: 8 beams x 1000 rows x 1024 x 24 caches, 1.08 GB with four
// distinct parents, 316 us with one float4 a thread and beam (too few bytes in
// flight for its waits), 217 with four, 168 (6.4 TB/s) with stores that pass the
// caches, too (one set of caches again and again; two in turn 210 to 229).
struct ReorderParams {
    LayerCaches caches;
    size_t beam_stride, count;  // floats; float4 of a beam's rows
    size_t start;               // floats of the rows before row0
    int32_t n_beams;
    const int32_t* parents;
};

template <int NB, int U>
__global__ __launch_bounds__(kCandThreads) void reorder_kernel(ReorderParams p) {
    typedef float vec __attribute__((ext_vector_type(4)));
    const size_t first = static_cast<size_t>(blockIdx.x) * U * kCandThreads + threadIdx.x;
    float* c = p.caches.c[blockIdx.y] + p.start;
    vec v[U][NB];
    int from[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int f = b < p.n_beams ? p.parents[b] : b;
        from[b] = f >= 0 && f < p.n_beams ? f : b;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const size_t i = first + u * kCandThreads;
        if (i < p.count)
#pragma unroll
            for (int b = 0; b < NB; ++b)
                if (from[b] != b)
                    v[u][b] = *reinterpret_cast<const vec*>(c + 4 * i + static_cast<size_t>(from[b]) * p.beam_stride);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const size_t i = first + u * kCandThreads;
        if (i < p.count)
#pragma unroll
            for (int b = 0; b < NB; ++b)
                if (from[b] != b)
                    __builtin_nontemporal_store(v[u][b],
                                                reinterpret_cast<vec*>(c + 4 * i + static_cast<size_t>(b) * p.beam_stride));
    }
}

// ---- beam search's selection ------------------------------------------------------
// score(b, v) = scores[b] + logits[b][v] - log sum_u e^logits[b][u]; the n_out
// best, ties to the lowest b vocab + v (Candidate).  Within a beam the order is the
// logits', so one pass over them leaves, per (beam, part of the vocabulary),
// the part's maximum, its sum of exponentials and its n_out best; a second
// kernel joins the parts in double, where candidates of different beams meet.
//
// Both find the n_out best of what their threads hold the same way.  The
// n_out-th largest of 256 maxima of disjoint groups is a threshold that at least
// n_out values reach, and few more: those go to LDS, and each one's rank is the
// number of better ones.  Where too many reach it (a vocabulary of equal
// logits), the best are taken one after another instead.
// Bound by the waits from step to step, not by bytes: 16 beams x 151936 words, 32
// out (9.7 MB), parts 9.6 us, 1.0 TB/s, and join 8.3 (11.4 with one thread, not
// eight, to rank a candidate); 4 x 32000, 8 out, 4.8 and 4.9.
struct SelectParams {
    const float* logits;
    const float* scores;
    const int32_t* finished;
    int32_t finished_token, n_beams, vocab, n_out, n_chunks;
    double2* ml;   // [beam][chunk] maximum, sum of e^(x - maximum)
    float2* best;  // [beam][chunk][n_out] logit, word (as bits), in falling order; -inf behind the last
    int32_t* out_parents;
    int32_t* out_tokens;
    float* out_scores;
};
constexpr int kGroups = 256;       // maxima that the threshold is taken from
constexpr int kMostRanked = 1024;  // values that are ranked

// NaN and -0 as -inf and +0
__device__ __forceinline__ float clean(float x) { return x != x ? -__builtin_inff() : x + 0.0f; }
// a float's bits in the floats' order, and back
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t o) {
    return __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
// Larger for the better candidate: the logit, then the lower word.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t word) {
    return static_cast<uint64_t>(ordered(x)) << 32 | ~word;
}

// A lower bound (its last 14 bits cleared) on the n-th largest of the 256 floats
// at maxima, by a wave: bit after bit of the ordered form, kept while n of them
// reach it.
__device__ __forceinline__ float nth_largest(const float* maxima, int n, int lane) {
    const float4 v = reinterpret_cast<const float4*>(maxima)[lane];
    const uint32_t o[4] = {ordered(v.x), ordered(v.y), ordered(v.z), ordered(v.w)};
    uint32_t least = 0;
    for (int bit = 31; bit >= 14; --bit) {
        const uint32_t t = least | 1u << bit;
        int count = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) count += __builtin_popcountll(__ballot(o[i] >= t));
        if (count >= n) least = t;
    }
    return least > 0x007fffffu ? unordered(least) : -__builtin_inff();  // (0x007fffff: -inf itself)
}

// The same of 64 floats, one a lane: a quarter of the counting, for few of them.
__device__ __forceinline__ float nth_of_wave(float v, int n) {
    const uint32_t o = ordered(v);
    uint32_t least = 0;
    for (int bit = 31; bit >= 14; --bit) {
        const uint32_t t = least | 1u << bit;
        if (__builtin_popcountll(__ballot(o >= t)) >= n) least = t;
    }
    return least > 0x007fffffu ? unordered(least) : -__builtin_inff();
}

__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
#pragma unroll
    for (int s = 32; s; s >>= 1) {
        const uint64_t o = __shfl_xor(v, s, 64);
        v = o > v ? o : v;
    }
    return v;
}

// The n_out best of the words that a work-group of T threads holds (thread tid's words: v0 +
// 4 T j + i), in two steps with a barrier between them: those that reach `least`
// (nth_largest's of the threads' maxima) go to LDS, held being 0 before a barrier, then
// the best go to `best` in falling order, -inf behind the last.  A NaN is no word, -0 is 0.
struct PartWords {  // (arrays of LDS: as one object they cost beam search 0.1 us)
    uint64_t (&keys)[kMostRanked];
    uint64_t* redk;  // a wave's
    int& held;
};
template <int V, int T>
__device__ __forceinline__ void gather_words(const float (&x)[V][4], int v0, float least, const PartWords& sh) {
    int mine = 0;
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) mine += x[j][i] >= least && x[j][i] > -__builtin_inff();
    if (mine) {
        int at = atomicAdd(&sh.held, mine);
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (x[j][i] >= least && x[j][i] > -__builtin_inff()) {
                    if (at < kMostRanked) sh.keys[at] = key_of(x[j][i] + 0.0f, static_cast<uint32_t>(v0 + 4 * T * j + i));
                    ++at;
                }
    }
}
template <int V, int T>
__device__ __forceinline__ void rank_words(const float (&x)[V][4], int v0, int n_out, float2* best, const PartWords& sh) {
    constexpr int kWavesHere = T / 64;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int n = sh.held;
    if (n <= kMostRanked) {
        for (int i = tid; i < n; i += T) {
            const uint64_t k = sh.keys[i];
            int rank = 0;
#pragma unroll 8
            for (int o = 0; o < n; ++o) rank += sh.keys[o] > k;
            if (rank < n_out)
                best[rank] = make_float2(unordered(static_cast<uint32_t>(k >> 32)),
                                         __builtin_bit_cast(float, ~static_cast<uint32_t>(k)));
        }
        for (int i = n + tid; i < n_out; i += T) best[i] = make_float2(-__builtin_inff(), 0.0f);
        return;
    }
    uint64_t last = ~uint64_t{0};
    for (int r = 0; r < n_out; ++r) {
        uint64_t k = 0;
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint64_t o = key_of(x[j][i] + 0.0f, static_cast<uint32_t>(v0 + 4 * T * j + i));
                if (x[j][i] > -__builtin_inff() && o < last && o > k) k = o;
            }
        k = wave_max_u64(k);
        __syncthreads();
        if (lane == 0) sh.redk[wv] = k;
        __syncthreads();
        k = sh.redk[0];
#pragma unroll
        for (int w = 1; w < kWavesHere; ++w) k = sh.redk[w] > k ? sh.redk[w] : k;
        if (tid == 0)
            best[r] = make_float2(k ? unordered(static_cast<uint32_t>(k >> 32)) : -__builtin_inff(),
                                  __builtin_bit_cast(float, ~static_cast<uint32_t>(k)));
        last = k;
    }
}

// A work-group holds 1024 V words of one beam in registers.
template <int V>
__global__ __launch_bounds__(kCandThreads) void select_parts_kernel(SelectParams p) {
    typedef float float4a4 __attribute__((ext_vector_type(4), aligned(4)));
    constexpr int kWavesHere = kCandThreads / 64;
    __shared__ __align__(16) float maxima[kGroups];
    __shared__ double sums[kWavesHere];
    __shared__ uint64_t keys[kMostRanked];
    __shared__ uint64_t redk[kCandThreads / 64];
    __shared__ int held;
    const PartWords sh{keys, redk, held};
    const int b = blockIdx.y, c = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    if (p.finished && p.finished[b]) return;
    const int v0 = c * 1024 * V + 4 * tid;  // this thread's words: v0 + 1024 j + i
    const float* row = p.logits + static_cast<size_t>(b) * p.vocab;
    float x[V][4], most = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int at = v0 + 1024 * j;
        if (at + 4 <= p.vocab) {
            const float4a4 w = *reinterpret_cast<const float4a4*>(row + at);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[j][i] = w[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[j][i] = at + i < p.vocab ? row[at + i] : -__builtin_inff();
        }
    }
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[j][i] = clean(x[j][i]);
            most = fmaxf(most, x[j][i]);
        }
    maxima[tid] = most;
    if (tid == 0) sh.held = 0;
    __syncthreads();
    // (the first maximum of the search is the part's)
    float m;
    {
        const float4 w = reinterpret_cast<const float4*>(maxima)[lane];
        m = wave_max(fmaxf(fmaxf(w.x, w.y), fmaxf(w.z, w.w)));
    }
    // exponentials of 32 bits, summed in 64 (a sum of 32 loses those of a large vocabulary
    // one by one beside a word that has most of the weight)
    double l = 0.0;
    if (m > -__builtin_inff())
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float e[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] = x[j][i] == m ? 1.0f : expf(x[j][i] - m);  // (x == m: an infinite maximum)
            l += (static_cast<double>(e[0]) + e[1]) + (static_cast<double>(e[2]) + e[3]);
        }
    l = wave_sum_f64(l);
    if (lane == 0) sums[wv] = l;
    const float least = nth_largest(maxima, p.n_out, lane);
    gather_words<V, kCandThreads>(x, v0, least, sh);
    __syncthreads();
    const size_t part = static_cast<size_t>(b) * p.n_chunks + c;
    float2* best = p.best + part * p.n_out;
    if (tid == 0) {
        double s = sums[0];
#pragma unroll
        for (int w = 1; w < kWavesHere; ++w) s += sums[w];
        p.ml[part] = make_double2(m, s);
    }
    rank_words<V, kCandThreads>(x, v0, p.n_out, best, sh);
}

// The order of equal scores: the lower beam, then the larger logit (64 bits may not
// part the scores of two logits, and the parts' lists are by logits), then the lower
// word.  Words are below 2^22, beams below 2^5.
constexpr int kWordBits = 22;
static_assert(kMaxBeamVocab <= 1 << kWordBits && kMaxBeams <= 1 << (63 - 32 - kWordBits));
__device__ __forceinline__ int64_t place_of(int beam, float logit, int word) {
    return static_cast<int64_t>(beam) << (32 + kWordBits) | static_cast<int64_t>(~ordered(logit)) << kWordBits | word;
}
struct Candidate {
    double score;
    int64_t at;  // place_of
    __device__ bool before(const Candidate& o) const { return score > o.score || (score == o.score && at < o.at); }
};

constexpr int kJoinThreads = 1024;
__global__ __launch_bounds__(kJoinThreads) void select_join_kernel(SelectParams p) {
    constexpr int kWavesHere = kJoinThreads / 64;
    __shared__ double base[kMaxBeams];  // scores[b] - log sum; -inf for a beam with nothing left
    __shared__ float top[kMaxBeams];
    __shared__ bool ended[kMaxBeams];   // (finished and scores may be among the outputs)
    __shared__ __align__(16) float maxima[kGroups];
    __shared__ Candidate ranked[kMostRanked];
    __shared__ int held;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const double inf = __builtin_inf();
    // entries of a part that the threshold is taken from: 2^shift
    const int parts = p.n_beams * p.n_chunks;
    int shift = 0;
    while (parts << shift < kGroups && 1 << shift < p.n_out) ++shift;
    const int first = 1 << shift;
    if (tid == 0) held = 0;
    // (read ahead of what needs the beams' sums)
    float2 ahead = make_float2(-__builtin_inff(), 0.0f);
    if (tid < kGroups && tid < parts << shift && (tid & first - 1) < p.n_out)
        ahead = p.best[static_cast<size_t>(tid >> shift) * p.n_out + (tid & first - 1)];
    // a wave per beam: the parts' maxima and sums
    for (int b = wv; b < p.n_beams; b += kWavesHere) {
        const float s = clean(p.scores[b]);
        const bool done = p.finished && p.finished[b];
        float m = -__builtin_inff();
        double sum = 0.0;
        if (!done) {
            const double2* ml = p.ml + static_cast<size_t>(b) * p.n_chunks;
            for (int c = lane; c < p.n_chunks; c += 64) m = fmaxf(m, static_cast<float>(ml[c].x));
            m = wave_max(m);
            for (int c = lane; c < p.n_chunks; c += 64) {
                const double2 v = ml[c];
                if (v.x > -__builtin_inff()) sum += v.y * (v.x == m ? 1.0 : exp(v.x - m));
            }
            sum = wave_sum_f64(sum);
        }
        if (lane == 0) {
            top[b] = m;
            ended[b] = done;
            base[b] = done ? s : m > -__builtin_inff() ? static_cast<double>(s) - log(sum) : -inf;
        }
    }
    __syncthreads();
    // the r-th best candidate of a part; -inf behind the last, and for a score that
    // the output's 32 bits hold as -inf
    auto entry = [&](int part, int r, float2 e) {
        const int b = part / p.n_chunks;
        if (ended[b])
            return r || part % p.n_chunks ? Candidate{-inf, 0}
                                          : Candidate{base[b], place_of(b, 0.0f, p.finished_token)};
        if (!(e.x > -__builtin_inff())) return Candidate{-inf, 0};
        const double score = base[b] + (e.x == top[b] ? 0.0 : static_cast<double>(e.x) - static_cast<double>(top[b]));
        if (!(static_cast<float>(score) > -__builtin_inff())) return Candidate{-inf, 0};
        return Candidate{score, place_of(b, e.x, __builtin_bit_cast(int32_t, e.y))};
    };
    auto candidate = [&](int part, int r) { return entry(part, r, p.best[static_cast<size_t>(part) * p.n_out + r]); };
    // The parts' lists fall, so the threshold comes from their first entries (as
    // many of each as make kGroups), and a list is read on only while it stays
    // above.  A score's float is in the scores' order, so floats serve.
    if (tid < kGroups) {
        float most = tid < parts << shift && (tid & first - 1) < p.n_out
                         ? static_cast<float>(entry(tid >> shift, tid & first - 1, ahead).score)
                         : -__builtin_inff();
        for (int j = tid + kGroups; j < parts << shift; j += kGroups)
            if ((j & first - 1) < p.n_out)
                most = fmaxf(most, static_cast<float>(candidate(j >> shift, j & first - 1).score));
        maxima[tid] = most;
    }
    __syncthreads();
    const float least = nth_largest(maxima, p.n_out, lane);
    // (eight entries of a list at once, and on from there one by one)
    const int wide = max(shift, 3), batch = 1 << wide;
    for (int j = tid; j < parts << wide; j += kJoinThreads)
        for (int r = j & batch - 1; r < p.n_out; ++r) {
            const Candidate c = candidate(j >> wide, r);
            if (!(c.score > -inf && static_cast<float>(c.score) >= least)) break;
            const int at = atomicAdd(&held, 1);
            if (at < kMostRanked) ranked[at] = c;
            if (r < batch - 1) break;
        }
    __syncthreads();
    auto write = [&](int i, const Candidate& c) {
        p.out_parents[i] = static_cast<int32_t>(c.at >> (32 + kWordBits));
        p.out_tokens[i] = static_cast<int32_t>(c.at & ((1 << kWordBits) - 1));
        p.out_scores[i] = static_cast<float>(c.score);
    };
    auto write_none = [&](int i) {
        p.out_parents[i] = p.out_tokens[i] = -1;
        p.out_scores[i] = -__builtin_inff();
    };
    const int n = held;
    if (n <= kMostRanked) {
        // eight threads a candidate
        for (int i = tid / 8; i < n; i += kJoinThreads / 8) {
            const Candidate c = ranked[i];
            int rank = 0;
#pragma unroll 4
            for (int o = tid % 8; o < n; o += 8) rank += ranked[o].before(c);
#pragma unroll
            for (int d = 1; d < 8; d *= 2) rank += __shfl_xor(rank, d, 8);
            if (tid % 8 == 0 && rank < p.n_out) write(rank, c);
        }
        for (int i = n + tid; i < p.n_out; i += kJoinThreads) write_none(i);
        return;
    }
    Candidate last{inf, -1};
    for (int r = 0; r < p.n_out; ++r) {
        Candidate mine{-inf, INT64_MAX};
        for (int j = tid; j < parts * p.n_out; j += kJoinThreads) {
            const Candidate c = candidate(j / p.n_out, j % p.n_out);
            if (c.score > -inf && last.before(c) && c.before(mine)) mine = c;
        }
#pragma unroll
        for (int s = 32; s; s >>= 1) {
            const Candidate o{__shfl_xor(mine.score, s, 64), __shfl_xor(mine.at, s, 64)};
            if (o.before(mine)) mine = o;
        }
        __syncthreads();
        if (lane == 0) ranked[wv] = mine;
        __syncthreads();
        last = ranked[0];
        for (int w = 1; w < kWavesHere; ++w)
            if (ranked[w].before(last)) last = ranked[w];
        if (tid == 0) write(r, last);
    }
}

// float4 of a thread (a work-group takes 1024 times as many words): the fewest
// that leave 512 parts, so that the second kernel has little to read (16 x 151936:
// 304 parts 9.2 + 8.2 us, 608 of half the size 8.1 + 9.9)
int32_t select_vectors(int32_t n_beams, int32_t vocab) {
    int32_t v = 2;
    while (v < 16 && static_cast<int64_t>(n_beams) * ((vocab + 1024 * v - 1) / (1024 * v)) > 512) v *= 2;
    return v;
}

// ---- log probabilities ----------------------------------------------------------------
// log p(v) = x_v - m - log S and H = log S - T / S, with S the sum of e^(x - m) and T that
// of e^(x - m) (x - m).  As in beam search's selection, a work-group holds a part of
// a row in registers and leaves its maximum, its two sums and its n_top best; a second
// kernel joins the parts of a row.  A row of one part is finished by the first.  Bound by
// reading the logits where rows are many (1999 x 32000 without alternatives 49 us, 5.2 TB/s of
// 256 MB), by the parts' chain of maximum, sums, threshold and ranking where alternatives are
// asked for (64 x 151936, 20 best: 15.5 and 5.6 us, 39 MB), by two launches and their
// latencies for one row (4.4 and 5.4).
struct LogprobParams {
    const float* logits;
    const int32_t* tokens;  // null: no out_logprobs
    int32_t vocab, n_top, n_chunks;
    double* sums;  // [row][chunk][3] maximum, S, T
    float2* best;  // [row][chunk][n_top] logit, word (as bits), in falling order; -inf behind the last
    float* out_logprobs;
    float* out_entropy;
    int32_t* out_top_tokens;
    float* out_top_logprobs;
};

// A row's log probabilities from its maximum and sums
struct RowSums {
    float m;
    double log_s;
    __device__ float logprob(float x) const {
        if (!(x > -__builtin_inff())) return -__builtin_inff();
        return static_cast<float>((x == m ? 0.0 : static_cast<double>(x) - static_cast<double>(m)) - log_s);
    }
};
// -inf without a token within the vocabulary
__device__ __forceinline__ float logit_of_token(const LogprobParams& p, size_t row) {
    const int32_t w = p.tokens ? p.tokens[row] : -1;
    return w >= 0 && w < p.vocab ? clean(p.logits[row * p.vocab + w]) : -__builtin_inff();
}
__device__ __forceinline__ void finish_row(const LogprobParams& p, size_t row, const RowSums& r, double s, double t,
                                           float token_logit) {
    if (p.tokens) p.out_logprobs[row] = r.logprob(token_logit);
    if (p.out_entropy) p.out_entropy[row] = s > 0.0 ? static_cast<float>(r.log_s - t / s) : 0.0f;
}
__device__ __forceinline__ void finish_top(const LogprobParams& p, size_t row, const RowSums& r, int i, float2 e) {
    const bool in = e.x > -__builtin_inff();
    p.out_top_tokens[row * p.n_top + i] = in ? __builtin_bit_cast(int32_t, e.y) : -1;
    p.out_top_logprobs[row * p.n_top + i] = r.logprob(e.x);
}

// e^d for d <= 8, off by two steps and by 2^-24 |d| of it (its argument in base 2 is rounded to
// 24 bits): log2(e) in two parts, as one of 24 bits would add d 2^-26.  (expf, with its range
// and special cases, 1999 rows of 32000: 60 us, not 51.)
__device__ __forceinline__ float exp_of(float d) {
    return __builtin_amdgcn_exp2f(fmaf(d, 1.44269502f, d * 1.92596299e-8f));
}

template <int V, int T>
__global__ __launch_bounds__(T) void logprob_parts_kernel(LogprobParams p) {
    typedef float float4a4 __attribute__((ext_vector_type(4), aligned(4)));
    constexpr int kWavesHere = T / 64;
    __shared__ __align__(16) float maxima[T];
    __shared__ double sums[kWavesHere][2];
    __shared__ uint64_t keys[kMostRanked];
    __shared__ uint64_t redk[kWavesHere];
    __shared__ int held;
    const PartWords sh{keys, redk, held};
    __shared__ float2 tops[kMaxTopWords];
    const size_t b = blockIdx.x / p.n_chunks;
    const int c = blockIdx.x % p.n_chunks, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int v0 = c * 4 * T * V + 4 * tid;  // this thread's words: v0 + 4 T j + i
    const float* row = p.logits + b * p.vocab;
    float x[V][4], most = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int at = v0 + 4 * T * j;
        if (at + 4 <= p.vocab) {
            const float4a4 w = *reinterpret_cast<const float4a4*>(row + at);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[j][i] = w[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[j][i] = at + i < p.vocab ? row[at + i] : -__builtin_inff();
        }
    }
    // (a NaN is no maximum, and its exponential below that of -200)
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) most = fmaxf(most, x[j][i]);
    maxima[tid] = most;
    if (tid == 0) sh.held = 0;
    __syncthreads();
    float m;
    if constexpr (T == 64) {
        m = wave_max(most);
    } else {
        const float4 w = reinterpret_cast<const float4*>(maxima)[lane];
        m = wave_max(fmaxf(fmaxf(w.x, w.y), fmaxf(w.z, w.w)));
    }
    double s = 0.0, t = 0.0;
    const bool finite = fabsf(m) < __builtin_inff();
    if (m > -__builtin_inff())
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float e[4], f[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // (below -104 the exponential is 0; beside an infinite maximum all others' are)
                float d = fmaxf(x[j][i] - m, -200.0f);
                if (!finite) d = x[j][i] == m ? 0.0f : -200.0f;
                e[i] = exp_of(d);
                f[i] = e[i] * d;
            }
            s += (static_cast<double>(e[0]) + e[1]) + (static_cast<double>(e[2]) + e[3]);
            t += (static_cast<double>(f[0]) + f[1]) + (static_cast<double>(f[2]) + f[3]);
        }
    s = wave_sum_f64(s);
    t = wave_sum_f64(t);
    if (lane == 0) {
        sums[wv][0] = s;
        sums[wv][1] = t;
    }
    // (up to 32 of 64 groups of threads: 64 rows of 151936, 20 best, 22.8 -> 21.6 us)
    float least;
    if constexpr (T == 64) {
        least = nth_of_wave(most, p.n_top);
    } else if (p.n_top > 32) {
        least = nth_largest(maxima, p.n_top, lane);
    } else {
        const float4 w = reinterpret_cast<const float4*>(maxima)[lane];
        least = nth_of_wave(fmaxf(fmaxf(w.x, w.y), fmaxf(w.z, w.w)), p.n_top);
    }
    gather_words<V, T>(x, v0, least, sh);
    __syncthreads();
    const size_t part = blockIdx.x;
    const bool whole = p.n_chunks == 1;
    s = sums[0][0];
    t = sums[0][1];
#pragma unroll
    for (int w = 1; w < kWavesHere; ++w) {
        s += sums[w][0];
        t += sums[w][1];
    }
    const RowSums r{m, log(s)};
    if (tid == 0) {
        if (whole) {
            finish_row(p, b, r, s, t, logit_of_token(p, b));
        } else {
            p.sums[3 * part] = m;
            p.sums[3 * part + 1] = s;
            p.sums[3 * part + 2] = t;
        }
    }
    rank_words<V, T>(x, v0, p.n_top, whole ? tops : p.best + part * p.n_top, sh);
    if (!whole) return;
    __syncthreads();
    if (tid < p.n_top) finish_top(p, b, r, tid, tops[tid]);
}

// Without alternatives a thread runs through its words with a maximum of its own, moved
// only where it is passed by 8 (an exponential of up to e^8 does not hurt), so that a
// part may be a row of any length and takes few registers.
constexpr int kStreamVectors = 8;  // float4 in flight
template <int T>
__global__ __launch_bounds__(T) void logprob_stream_kernel(LogprobParams p, int32_t words) {
    typedef float float4a4 __attribute__((ext_vector_type(4), aligned(4)));
    constexpr int kWavesHere = T / 64;
    __shared__ double sums[kWavesHere][3];
    const size_t b = blockIdx.x / p.n_chunks;
    const int c = blockIdx.x % p.n_chunks, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int64_t first = static_cast<int64_t>(c) * words, end = first + words < p.vocab ? first + words : p.vocab;
    const float* row = p.logits + b * p.vocab;
    float m = -__builtin_inff();
    double s = 0.0, t = 0.0;
    for (int64_t at0 = first + 4 * tid; at0 < end; at0 += 4 * T * kStreamVectors) {
        float x[kStreamVectors][4], most = -__builtin_inff();
#pragma unroll
        for (int j = 0; j < kStreamVectors; ++j) {
            const int64_t at = at0 + 4 * T * j;
            if (at + 4 <= end) {
                const float4a4 w = *reinterpret_cast<const float4a4*>(row + at);
#pragma unroll
                for (int i = 0; i < 4; ++i) x[j][i] = w[i];
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) x[j][i] = at + i < end ? row[at + i] : -__builtin_inff();
            }
        }
        // (a NaN is no maximum, and its exponential below that of -200)
#pragma unroll
        for (int j = 0; j < kStreamVectors; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) most = fmaxf(most, x[j][i]);
        if (most > m + 8.0f) {
            if (s > 0.0) {
                const double d = static_cast<double>(m) - static_cast<double>(most), f = exp(d);
                t = f > 0.0 ? f * (t + d * s) : 0.0;
                s *= f;
            }
            m = most;
        }
        const bool finite = fabsf(m) < __builtin_inff();
#pragma unroll
        for (int j = 0; j < kStreamVectors; ++j) {
            float e[4], f[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // (below -104 the exponential is 0; beside an infinite maximum all others' are)
                float d = fmaxf(x[j][i] - m, -200.0f);
                if (!finite) d = x[j][i] == m && m > 0.0f ? 0.0f : -200.0f;
                e[i] = exp_of(d);
                f[i] = e[i] * d;
            }
            s += (static_cast<double>(e[0]) + e[1]) + (static_cast<double>(e[2]) + e[3]);
            t += (static_cast<double>(f[0]) + f[1]) + (static_cast<double>(f[2]) + f[3]);
        }
    }
    // the threads' sums to the wave's maximum, the waves' to the work-group's
    auto moved = [](double& s, double& t, float from, float to) {
        const double d = from == to ? 0.0 : static_cast<double>(from) - static_cast<double>(to), f = exp(d);
        t = f > 0.0 && s > 0.0 ? f * (t + d * s) : 0.0;
        s = s > 0.0 ? f * s : 0.0;
    };
    const float mw = wave_max(m);
    moved(s, t, m, mw);
    s = wave_sum_f64(s);
    t = wave_sum_f64(t);
    if (lane == 0 && T > 64) {
        sums[wv][0] = mw;
        sums[wv][1] = s;
        sums[wv][2] = t;
    }
    if (T > 64) __syncthreads();
    if (tid) return;
    float M = mw;
#pragma unroll
    for (int w = 1; w < kWavesHere; ++w) M = fmaxf(M, static_cast<float>(sums[w][0]));
    if (T > 64) {
        s = t = 0.0;
#pragma unroll
        for (int w = 0; w < kWavesHere; ++w) {
            double ws = sums[w][1], wt = sums[w][2];
            moved(ws, wt, static_cast<float>(sums[w][0]), M);
            s += ws;
            t += wt;
        }
    }
    if (p.n_chunks == 1) {
        finish_row(p, b, RowSums{M, log(s)}, s, t, logit_of_token(p, b));
    } else {
        double* to = p.sums + 3 * static_cast<size_t>(blockIdx.x);
        to[0] = M;
        to[1] = s;
        to[2] = t;
    }
}

__global__ __launch_bounds__(kCandThreads) void logprob_join_kernel(LogprobParams p) {
    __shared__ __align__(16) float maxima[kGroups];
    __shared__ uint64_t keys[kMostRanked];
    __shared__ uint64_t redk[kCandThreads / 64];
    __shared__ int held;
    const PartWords sh{keys, redk, held};
    const size_t row = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, parts = p.n_chunks;
    const double* sums = p.sums + 3 * row * parts;
    const float2* best = p.best + row * parts * p.n_top;
    // (read ahead of what needs the sums: the first entries of the parts' lists, and the token's logit)
    int shift = 0;
    while (parts << shift < kGroups && 1 << shift < p.n_top) ++shift;
    const int first = 1 << shift;
    float most = -__builtin_inff();
    for (int j = tid; j < parts << shift; j += kGroups)
        if ((j & (first - 1)) < p.n_top) most = fmaxf(most, best[static_cast<size_t>(j >> shift) * p.n_top + (j & (first - 1))].x);
    const float token_logit = logit_of_token(p, row);
    // every wave: the parts' maxima and sums
    float m = -__builtin_inff();
    for (int c = lane; c < parts; c += 64) m = fmaxf(m, static_cast<float>(sums[3 * c]));
    m = wave_max(m);
    double s = 0.0, t = 0.0;
    for (int c = lane; c < parts; c += 64) {
        const double mc = sums[3 * c];
        if (mc > -__builtin_inff()) {
            const double d = mc == m ? 0.0 : mc - m, f = exp(d);
            s += f * sums[3 * c + 1];
            t += f * (sums[3 * c + 2] + (f > 0.0 ? d * sums[3 * c + 1] : 0.0));
        }
    }
    s = wave_sum_f64(s);
    t = wave_sum_f64(t);
    const RowSums r{m, log(s)};
    if (tid == 0) {
        finish_row(p, row, r, s, t, token_logit);
        sh.held = 0;
    }
    if (p.n_top == 0) return;
    // The parts' lists fall: a threshold from their first 2^shift entries, and a list
    // is read on only while it stays above.
    maxima[tid] = most;
    __syncthreads();
    const float least = nth_largest(maxima, p.n_top, lane);
    const int wide = max(shift, 3), batch = 1 << wide;
    for (int j = tid; j < parts << wide; j += kCandThreads)
        for (int i = j & (batch - 1); i < p.n_top; ++i) {
            const float2 e = best[static_cast<size_t>(j >> wide) * p.n_top + i];
            if (!(e.x > -__builtin_inff() && e.x >= least)) break;
            const int at = atomicAdd(&sh.held, 1);
            if (at < kMostRanked) sh.keys[at] = key_of(e.x, __builtin_bit_cast(uint32_t, e.y));
            if (i < batch - 1) break;
        }
    __syncthreads();
    auto word_of = [](uint64_t k) {
        return make_float2(unordered(static_cast<uint32_t>(k >> 32)), __builtin_bit_cast(float, ~static_cast<uint32_t>(k)));
    };
    const int n = sh.held;
    if (n <= kMostRanked) {
        // eight threads a candidate
        for (int i = tid / 8; i < n; i += kCandThreads / 8) {
            const uint64_t k = sh.keys[i];
            int rank = 0;
#pragma unroll 4
            for (int o = tid % 8; o < n; o += 8) rank += sh.keys[o] > k;
#pragma unroll
            for (int d = 1; d < 8; d *= 2) rank += __shfl_xor(rank, d, 8);
            if (tid % 8 == 0 && rank < p.n_top) finish_top(p, row, r, rank, word_of(k));
        }
        for (int i = n + tid; i < p.n_top; i += kCandThreads) finish_top(p, row, r, i, make_float2(-__builtin_inff(), 0.0f));
        return;
    }
    uint64_t last = ~uint64_t{0};
    for (int i = 0; i < p.n_top; ++i) {
        uint64_t k = 0;
        for (int j = tid; j < parts * p.n_top; j += kCandThreads) {
            const float2 e = best[j];
            const uint64_t o = key_of(e.x, __builtin_bit_cast(uint32_t, e.y));
            if (e.x > -__builtin_inff() && o < last && o > k) k = o;
        }
        k = wave_max_u64(k);
        __syncthreads();
        if (lane == 0) sh.redk[wv] = k;
        __syncthreads();
        k = sh.redk[0];
#pragma unroll
        for (int w = 1; w < kCandThreads / 64; ++w) k = sh.redk[w] > k ? sh.redk[w] : k;
        if (tid == 0) finish_top(p, row, r, i, k ? word_of(k) : make_float2(-__builtin_inff(), 0.0f));
        last = k;
    }
}

// Rows of so few words are a wave's (20000 x 300 72 -> 28 us, with 3 alternatives 55 -> 28;
// 4000 x 1000 22.1 -> 9.3, with 20 16.7 -> 11.0), unless more than 32 of 64 lanes' maxima would
// make their threshold (64 x 1000, 64 alternatives: 61 us, not 7.7)
constexpr int32_t kWaveWords = 1024;
// Words of a part: the most that leave 1024 parts over all rows, up to a row without
// alternatives, else what leaves four work-groups a CU their registers (20 alternatives, 4096,
// 8192 and 16384 words: 64 x 151936 22.1, 21.5, 25.4 us; 128 x 151936 32.0, 29.8, 37.9; 2000 x
// 32000 84, 75, 95).
int32_t logprob_words(int32_t n_rows, int32_t vocab, int32_t n_top) {
    const int32_t most = n_top ? 8192 : kMaxBeamVocab;
    int32_t w = 2048;
    while (w < most && w < vocab && static_cast<int64_t>(n_rows) * ((vocab + 2 * w - 1) / (2 * w)) >= 1024) w *= 2;
    return w;
}

template <class F>
hipError_t by_layers(float* const* k, float* const* v, int32_t n_layers, F&& launch) {
    for (int32_t l0 = 0; l0 < n_layers; l0 += kLayerGroup) {
        const int32_t n = n_layers - l0 < kLayerGroup ? n_layers - l0 : kLayerGroup;
        LayerCaches c{};
        for (int32_t l = 0; l < n; ++l) {
            c.c[2 * l] = k[l0 + l];
            c.c[2 * l + 1] = v[l0 + l];
        }
        launch(c, 2 * n);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace

hipError_t launch_kv_keep_rows(float* const* k, float* const* v, int32_t n_layers, int32_t kv_dim, int32_t row0,
                               const int32_t* rows, int32_t n, hipStream_t stream) {
    if (n < 0 || n > kMaxKeepRows || kv_dim < 4 || kv_dim % 4 || row0 < 0) return hipErrorInvalidValue;
    int32_t stay = 0;
    while (stay < n && rows[stay] == stay) ++stay;
    if (stay == n) return hipSuccess;
    KeepParams p{};
    p.kv_dim = kv_dim;
    p.n = n - stay;
    p.row0 = static_cast<size_t>(row0) + stay;
    for (int32_t i = stay; i < n; ++i) p.rows[i - stay] = static_cast<uint16_t>(rows[i] - stay);
    // one float a thread while that leaves fewer than 4096 waves (a wave's loads
    // are then whole 256-byte lines of a row), else four
    const bool narrow = static_cast<int64_t>(n_layers) * 2 * ((kv_dim + 63) / 64) < 4096;
    const int32_t per = narrow ? 64 : 256;
    return by_layers(k, v, n_layers, [&](const LayerCaches& c, int32_t caches) {
        p.caches = c;
        const dim3 grid((kv_dim + per - 1) / per, caches);
        // (a call of few rows would read 48 for nothing)
        if (p.n <= 16 && narrow) hipLaunchKernelGGL((keep_rows_kernel<1, 16>), grid, dim3(64), 0, stream, p);
        else if (narrow) hipLaunchKernelGGL((keep_rows_kernel<1, 64>), grid, dim3(64), 0, stream, p);
        else if (p.n <= 16) hipLaunchKernelGGL((keep_rows_kernel<4, 16>), grid, dim3(64), 0, stream, p);
        else hipLaunchKernelGGL((keep_rows_kernel<4, 32>), grid, dim3(64), 0, stream, p);
    });
}

hipError_t launch_kv_reorder(float* const* k, float* const* v, int32_t n_layers, int32_t n_beams, size_t beam_stride,
                             int32_t kv_dim, int32_t row0, int32_t n_rows, const int32_t* parents,
                             hipStream_t stream) {
    if (n_beams < 1 || n_beams > kMaxBeams || kv_dim < 4 || kv_dim % 4 || beam_stride % 4 || row0 < 0 || n_rows < 0)
        return hipErrorInvalidValue;
    ReorderParams p{};
    p.beam_stride = beam_stride;
    p.count = static_cast<size_t>(n_rows) * kv_dim / 4;
    p.start = static_cast<size_t>(row0) * kv_dim;
    p.n_beams = n_beams;
    p.parents = parents;
    // float4 a thread and beam (128 registers hold 32 of them): one, two, four,
    // us: 8 beams x 1000 rows x 1024 x 24 caches 307, 187, 168; 8 x 100 x 72 caches
    // 58, 47, 48; 4 x 5 x 72 4.2, 3.4, 4.6; 8 x 10 rows of 512 x 8 (40 tiles) 4.2,
    // 8.0, 8.4
    const size_t tiles = (p.count + kCandThreads - 1) / kCandThreads, all = tiles * 2 * n_layers;
    const int32_t u = all < 256 || n_beams > 16 ? 1 : all < 16384 || n_beams > 8 ? 2 : 4;
    const size_t groups = (tiles + u - 1) / u;
    if (groups > 0x7fffffffu) return hipErrorInvalidValue;
    return by_layers(k, v, n_layers, [&](const LayerCaches& c, int32_t caches) {
        p.caches = c;
        const dim3 grid(static_cast<uint32_t>(groups), caches);
        if (n_beams <= 8 && u == 4) hipLaunchKernelGGL((reorder_kernel<8, 4>), grid, dim3(kCandThreads), 0, stream, p);
        else if (n_beams <= 8 && u == 2) hipLaunchKernelGGL((reorder_kernel<8, 2>), grid, dim3(kCandThreads), 0, stream, p);
        else if (n_beams <= 8) hipLaunchKernelGGL((reorder_kernel<8, 1>), grid, dim3(kCandThreads), 0, stream, p);
        else if (n_beams <= 16 && u == 2) hipLaunchKernelGGL((reorder_kernel<16, 2>), grid, dim3(kCandThreads), 0, stream, p);
        else hipLaunchKernelGGL((reorder_kernel<32, 1>), grid, dim3(kCandThreads), 0, stream, p);
    });
}

size_t beam_select_workspace_bytes(int32_t n_beams, int32_t vocab, int32_t n_out) {
    const int32_t words = 1024 * select_vectors(n_beams, vocab);
    return static_cast<size_t>(n_beams) * ((vocab + words - 1) / words) * (sizeof(double2) + sizeof(float2) * n_out);
}

hipError_t launch_beam_select(const float* logits, int32_t n_beams, int32_t vocab, const float* scores,
                              const int32_t* finished, int32_t finished_token, int32_t n_out, int32_t* out_parents,
                              int32_t* out_tokens, float* out_scores, void* workspace, size_t workspace_bytes,
                              hipStream_t stream) {
    if (n_beams < 1 || n_beams > kMaxBeams || vocab < 1 || vocab > kMaxBeamVocab || n_out < 1 || n_out > kMaxBeamOut ||
        workspace_bytes < beam_select_workspace_bytes(n_beams, vocab, n_out))
        return hipErrorInvalidValue;
    SelectParams p{};
    p.logits = logits;
    p.scores = scores;
    p.finished = finished;
    p.finished_token = finished_token;
    p.n_beams = n_beams;
    p.vocab = vocab;
    p.n_out = n_out;
    const int32_t v = select_vectors(n_beams, vocab);
    p.n_chunks = (vocab + 1024 * v - 1) / (1024 * v);
    p.ml = static_cast<double2*>(workspace);
    p.best = reinterpret_cast<float2*>(p.ml + static_cast<size_t>(n_beams) * p.n_chunks);
    p.out_parents = out_parents;
    p.out_tokens = out_tokens;
    p.out_scores = out_scores;
    const dim3 grid(p.n_chunks, n_beams);
    if (v == 2) hipLaunchKernelGGL(select_parts_kernel<2>, grid, dim3(kCandThreads), 0, stream, p);
    else if (v == 4) hipLaunchKernelGGL(select_parts_kernel<4>, grid, dim3(kCandThreads), 0, stream, p);
    else if (v == 8) hipLaunchKernelGGL(select_parts_kernel<8>, grid, dim3(kCandThreads), 0, stream, p);
    else hipLaunchKernelGGL(select_parts_kernel<16>, grid, dim3(kCandThreads), 0, stream, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(select_join_kernel, dim3(1), dim3(kJoinThreads), 0, stream, p);
    return hipGetLastError();
}

size_t token_logprobs_workspace_bytes(int32_t n_rows, int32_t vocab, int32_t n_top) {
    const int32_t words = logprob_words(n_rows, vocab, n_top), chunks = (vocab + words - 1) / words;
    return chunks == 1 ? 0 : static_cast<size_t>(n_rows) * chunks * (3 * sizeof(double) + sizeof(float2) * n_top);
}

hipError_t launch_token_logprobs(const float* logits, int32_t n_rows, int32_t vocab, const int32_t* tokens,
                                 int32_t n_top, float* out_logprobs, float* out_entropy, int32_t* out_top_tokens,
                                 float* out_top_logprobs, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    if (n_rows < 1 || vocab < 1 || vocab > kMaxBeamVocab || n_top < 0 || n_top > kMaxTopWords ||
        workspace_bytes < token_logprobs_workspace_bytes(n_rows, vocab, n_top))
        return hipErrorInvalidValue;
    const int32_t words = logprob_words(n_rows, vocab, n_top);
    const int32_t n_chunks = (vocab + words - 1) / words;
    const int64_t parts = static_cast<int64_t>(n_rows) * n_chunks;
    if (parts > 0x7fffffff) return hipErrorInvalidValue;
    double* const sums = static_cast<double*>(workspace);
    float2* const best = reinterpret_cast<float2*>(sums + 3 * parts);
    // (rows whose parts are one launch's work-groups)
    const int32_t at_once = std::max(1, (1 << 22) / n_chunks);
    for (int64_t r0 = 0; r0 < n_rows; r0 += at_once) {
        const int32_t rows = static_cast<int32_t>(std::min<int64_t>(at_once, n_rows - r0));
        LogprobParams p{};
        p.logits = logits + r0 * vocab;
        p.tokens = tokens ? tokens + r0 : nullptr;
        p.vocab = vocab;
        p.n_top = n_top;
        p.n_chunks = n_chunks;
        p.sums = sums + 3 * r0 * n_chunks;
        p.best = best + r0 * n_chunks * n_top;
        p.out_logprobs = out_logprobs ? out_logprobs + r0 : nullptr;
        p.out_entropy = out_entropy ? out_entropy + r0 : nullptr;
        p.out_top_tokens = out_top_tokens ? out_top_tokens + r0 * n_top : nullptr;
        p.out_top_logprobs = out_top_logprobs ? out_top_logprobs + r0 * n_top : nullptr;
        const dim3 grid(static_cast<uint32_t>(rows) * n_chunks);
        const dim3 block(kCandThreads), wave(64);
        if (n_top == 0 && vocab <= kWaveWords) hipLaunchKernelGGL(logprob_stream_kernel<64>, grid, wave, 0, stream, p, words);
        else if (n_top == 0) hipLaunchKernelGGL(logprob_stream_kernel<kCandThreads>, grid, block, 0, stream, p, words);
        else if (vocab <= kWaveWords && n_top <= 32) hipLaunchKernelGGL((logprob_parts_kernel<kWaveWords / 256, 64>), grid, wave, 0, stream, p);
        else if (words == 2048) hipLaunchKernelGGL((logprob_parts_kernel<2, kCandThreads>), grid, block, 0, stream, p);
        else if (words == 4096) hipLaunchKernelGGL((logprob_parts_kernel<4, kCandThreads>), grid, block, 0, stream, p);
        else hipLaunchKernelGGL((logprob_parts_kernel<8, kCandThreads>), grid, block, 0, stream, p);
        hipError_t e = hipGetLastError();
        if (e == hipSuccess && n_chunks > 1) {
            hipLaunchKernelGGL(logprob_join_kernel, dim3(rows), dim3(kCandThreads), 0, stream, p);
            e = hipGetLastError();
        }
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace gncx
