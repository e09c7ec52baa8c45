// attention.hip -- GQA/MQA/SWA decode attention step for gfx950.
//
// Semantics of the reference's gncx_mqa_attention_step_ext
// (csrc/gncx_llm_kernels.cpp:1887-1994): optionally store k_new/v_new at row
// `pos` of the layer's KV cache, then for every query head h (KV head
// h / (n_heads / n_kv_heads)) softmax((q . k_t) * scale) over the window
// [max(0, pos - sw + 1), pos] and o = sum_t p_t v_t with the reference's
// normaliser 1 / (sum + 1e-12).
//
// MI355X design (flash-decoding): the window is cut into chunks; one
// work-group owns (KV head, chunk) and serves all query heads of its group, so
// each KV row is read from HBM once (the reference re-reads it per query
// head).  A token row of one KV head is read by hd/16 lanes with coalesced
// 16-byte loads; scores go to LDS, each wave reduces one head's max/sum, the
// V pass accumulates in registers and the waves combine through LDS.  A
// second small kernel merges the chunk partials with the log-sum-exp rule.
//
// Optional fused prologue (cpp:895-953 per-head RMSNorm, then cpp:1797-1862
// NEOX RoPE with a host-computed cos/sin table) is applied to q and k_new in
// LDS before the scan, with the same arithmetic as the stand-alone kernels.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>
#include <vector>

#include "gncx_device.h"
#include "gncx_launch.h"

namespace gncx {
namespace {

using namespace dev;

typedef float floatx16 __attribute__((ext_vector_type(16)));

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kHeadBlock = 4;     // query heads handled per pass (one wave each in the softmax)
constexpr int kMaxChunk = 1024;   // tokens per work-group
// Work-groups a call aims for: windows that fit 32-token chunks at kTargetGroups
// keep those (one pass per work-group, K/V loaded up front); longer windows
// take about half as many, longer chunks.  Measured per call, GQA 32/8 x 128
// (chunk + merge), 1024 / 512 target work-groups: ctx 2100: 13.8 / 18.0 us;
// ctx 4096: 16.1 / 17.3; ctx 8192: 27.6 / 26.5; ctx 16384: 42.5 / 34.5;
// ctx 32768: 63.2 / 56.4; ctx 65536: 110 / 101; GQA 32/4 ctx 32768: 60.7 /
// 52.6 us.
constexpr int kTargetGroups = 1024;
constexpr int kTargetGroupsLong = 512;

struct AttnParams {
    const float* q;
    const float* k_new;
    const float* v_new;
    float* k_cache;
    float* v_cache;
    float* part_o;  // [n_split][n_heads][hd]
    float* part_ml; // [n_split][n_heads][2]  (max, sum)
    float* q_out;
    float* k_out;
    const float* q_gamma;
    const float* k_gamma;
    int32_t pos, n_heads, n_kv, t0, t1, chunk, use_new, norm_qk, has_rope;
    float scale, eps;
    RopeTable rope;
};


// The prologue's per-lane operands (norm weights of the elements a lane
// normalises, the RoPE rows of the pairs it rotates), loaded into registers
// with the other small operands before the K/V rows, so the prologue waits
// for no memory.
template <int HD>
struct ProRegs {
    static constexpr int NE = HD / 64 > 0 ? HD / 64 : 1;  // elements per lane
    static constexpr int NR = (HD / 2 + 63) / 64;         // rotated pairs per lane
    float gq[NE], gk[NE], c[NR], s[NR];
    // unconditional loads (a missing weight reads q, whose first HD values
    // exist, and is never used: has_gamma): with no load
    // behind a branch the compiler counts them exactly and waits for these
    // alone, not for the K/V rows issued after them
    __device__ __forceinline__ void load(const AttnParams& p, int lane) {
        const float* gqp = p.q_gamma ? p.q_gamma : p.q;
        const float* gkp = p.k_gamma ? p.k_gamma : p.q;
#pragma unroll
        for (int e = 0; e < NE; ++e) {
            const int i = lane + 64 * e < HD ? lane + 64 * e : 0;
            gq[e] = gqp[i];
            gk[e] = gkp[i];
        }
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const int i = lane + 64 * r < HD / 2 ? lane + 64 * r : 0;
            c[r] = p.rope.c[i];
            s[r] = p.rope.s[i];
        }
    }
};

// Per-head RMSNorm then RoPE of one head held in LDS, one wave, with the
// operands in registers; no weight without has_gamma
template <int HD>
__device__ __forceinline__ void prologue_head_r(float* v, const float* g, bool has_gamma, bool norm, bool rope,
                                                float eps, const ProRegs<HD>& pr, int lane) {
#pragma clang fp contract(off)
    if (norm) {
        const float inv = head_inv_rms(v, HD, eps, lane);
#pragma unroll
        for (int e = 0; e < ProRegs<HD>::NE; ++e) {
            const int i = lane + 64 * e;
            if (i < HD) {
                const float x = v[i] * inv;
                v[i] = has_gamma ? x * g[e] : x;
            }
        }
    }
    if (rope) {
        constexpr int H = HD / 2;
#pragma unroll
        for (int r = 0; r < ProRegs<HD>::NR; ++r) {
            const int i = lane + 64 * r;
            if (i < H) {
                const float x1 = v[i], x2 = v[i + H];
                v[i] = x1 * pr.c[r] - x2 * pr.s[r];
                v[i + H] = x2 * pr.c[r] + x1 * pr.s[r];
            }
        }
    }
}

// SHORT: the chunk fits one pass (chunk <= TPP tokens).  Each thread's K and V
// slices are then loaded at the start, ahead of q, so a work-group waits for
// HBM once instead of three times in a row (q, then K, then V after the
// softmax), and head blocks after the first re-read nothing.
template <int HD, bool SHORT>
__global__ __launch_bounds__(kThreads) void attn_chunk_kernel(AttnParams p) {
    constexpr int LPT = HD / 16;          // lanes per token row (16 dims each)
    constexpr int TPP = kThreads / LPT;   // tokens per pass
    extern __shared__ __align__(16) float smem[];
    const int G = p.n_heads / p.n_kv;
    float* sc = smem;                                   // [kHeadBlock][chunk]
    float* red = sc + kHeadBlock * p.chunk;             // [kWaves][kHeadBlock][HD]
    float* qs = red + kWaves * kHeadBlock * HD;         // [G][HD]  (prologue result)
    float* ks = qs + G * HD;                            // [HD]
    float* vs = ks + HD;                                // SHORT: [TPP][HD], the chunk's V rows

    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int hk = blockIdx.x;
    const int split = blockIdx.y;
    const int ta = p.t0 + split * p.chunk;
    const int tb = min(p.t1, ta + p.chunk);
    const int j = tid % LPT;       // 16-dim slice of the row
    const int ts = tid / LPT;      // token slot within a pass
    const size_t kv_dim = static_cast<size_t>(p.n_kv) * HD;
    const bool have_new = p.use_new != 0;

    // q rows of this KV head's query heads, k_new and the prologue operands
    // first: the prologue then runs while the K/V rows are still in flight.
    // Every early load is unconditional (indices clamped, pointers selected,
    // unused values replaced afterwards), so the compiler counts them exactly
    // and the prologue waits for these loads alone: a load behind a branch made
    // it wait for every load issued so far, the K/V rows included.
    constexpr int kQRegs = 8;  // q values per thread held across the K/V issue
    const int gq_n = G * HD;
    const float* qg = p.q + static_cast<size_t>(hk) * G * HD;
    float qreg[kQRegs];
#pragma unroll
    for (int u = 0; u < kQRegs; ++u) {
        const int i = tid + u * kThreads;
        qreg[u] = qg[i < gq_n ? i : gq_n - 1];
    }
    // without a new row, q (at least n_kv HD values) stands in for k_new
    const float* knp = have_new ? p.k_new : p.q;
    const float kreg = knp[static_cast<size_t>(hk) * HD + (tid < HD ? tid : 0)];  // used where have_new && tid < HD
    const bool pro = p.norm_qk || p.has_rope;
    ProRegs<HD> pr;
    if (pro) pr.load(p, lane);

    // SHORT: this thread's token is ta + ts; its K / V slices are loaded now
    // (the new token's K comes from LDS after the prologue, its V from v_new);
    // a slot past the chunk reads row ta, and neither its score nor its V row
    // is used
    // (native vectors: float4 copies are memcpys, and a V slice copied that
    // way went through scratch memory on its way to LDS)
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    float4 kpre[4];
    f32x4 vpre[4];
    const int tok0 = ta + ts;
    const bool valid0 = tok0 < tb;
    const bool new0 = have_new && tok0 == p.pos;
    if constexpr (SHORT) {
        const int tokc = valid0 ? tok0 : ta;
        const float* ksrc = p.k_cache + static_cast<size_t>(tokc) * kv_dim + static_cast<size_t>(hk) * HD;
        const float* vsrc = new0 ? p.v_new + static_cast<size_t>(hk) * HD
                                 : p.v_cache + static_cast<size_t>(tokc) * kv_dim + static_cast<size_t>(hk) * HD;
#pragma unroll
        for (int c = 0; c < 4; ++c) kpre[c] = *reinterpret_cast<const float4*>(ksrc + 4 * (j + LPT * c));
#pragma unroll
        for (int c = 0; c < 4; ++c) vpre[c] = *reinterpret_cast<const f32x4*>(vsrc + 4 * (j + LPT * c));
    }

    // ---- q (and k_new) into LDS, with the optional prologue ----
#pragma unroll
    for (int u = 0; u < kQRegs; ++u) {
        const int i = tid + u * kThreads;
        if (i < G * HD) qs[i] = qreg[u];
    }
    for (int i = tid + kQRegs * kThreads; i < G * HD; i += kThreads) qs[i] = qg[i];
    if (have_new && tid < HD) ks[tid] = kreg;
    __syncthreads();
    // The work-group whose chunk holds `pos` (the last one) is the only one
    // that reads the new k: it alone runs k's prologue and writes the
    // prologue results back to q_out / k_out.
    const bool owner = p.pos >= ta && p.pos < tb;
    if (pro) {
        for (int h = wv; h < G + (have_new && owner ? 1 : 0); h += kWaves) {
            if (h < G) prologue_head_r<HD>(qs + h * HD, pr.gq, p.q_gamma != nullptr, p.norm_qk, p.has_rope, p.eps, pr, lane);
            else prologue_head_r<HD>(ks, pr.gk, p.k_gamma != nullptr, p.norm_qk, p.has_rope, p.eps, pr, lane);
        }
        __syncthreads();
        if (owner) {
            if (p.q_out)
                for (int i = tid; i < G * HD; i += kThreads) p.q_out[static_cast<size_t>(hk) * G * HD + i] = qs[i];
            if (p.k_out && have_new)
                for (int i = tid; i < HD; i += kThreads) p.k_out[static_cast<size_t>(hk) * HD + i] = ks[i];
        }
    }
    // the work-group whose chunk holds `pos` stores the new K/V row of its head
    if (have_new && p.pos >= ta && p.pos < tb) {
        float* kd = p.k_cache + static_cast<size_t>(p.pos) * kv_dim + static_cast<size_t>(hk) * HD;
        float* vd = p.v_cache + static_cast<size_t>(p.pos) * kv_dim + static_cast<size_t>(hk) * HD;
        const float* vn = p.v_new + static_cast<size_t>(hk) * HD;
        for (int i = tid; i < HD; i += kThreads) {
            kd[i] = ks[i];
            vd[i] = vn[i];
        }
    }

    // SHORT: the chunk's V rows into LDS for pass 2 (their last use of
    // registers: held across the head-block loop they went to scratch memory)
    if constexpr (SHORT) {
#pragma unroll
        for (int c = 0; c < 4; ++c) *reinterpret_cast<f32x4*>(vs + ts * HD + 4 * (j + LPT * c)) = vpre[c];
    }

    for (int hb = 0; hb < G; hb += kHeadBlock) {
        const int nh = min(kHeadBlock, G - hb);
        // q slices of this lane: kept in registers across the token passes of
        // a long chunk; a one-pass chunk reads each head's slices from LDS where
        // it uses them (64 registers fewer: four work-groups per CU)
        float4 qf[SHORT ? 1 : kHeadBlock][4];
        if constexpr (!SHORT) {
#pragma unroll
            for (int h = 0; h < kHeadBlock; ++h)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    qf[h][c] = h < nh ? *reinterpret_cast<const float4*>(qs + (hb + h) * HD + 4 * (j + LPT * c))
                                      : make_float4(0.f, 0.f, 0.f, 0.f);
        }

        // ---- pass 1: scores ----
        for (int t = ta; t < tb; t += TPP) {
            const int tok = t + ts;
            const bool valid = tok < tb;
            float4 kf[4];
            if (SHORT) {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    kf[c] = new0 ? *reinterpret_cast<const float4*>(ks + 4 * (j + LPT * c)) : kpre[c];
            } else if (valid) {
                const float* src = (have_new && tok == p.pos)
                                       ? ks
                                       : p.k_cache + static_cast<size_t>(tok) * kv_dim + static_cast<size_t>(hk) * HD;
#pragma unroll
                for (int c = 0; c < 4; ++c) kf[c] = *reinterpret_cast<const float4*>(src + 4 * (j + LPT * c));
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c) kf[c] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int h = 0; h < kHeadBlock; ++h) {
                float s = 0.0f;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float4 qv;
                    if constexpr (SHORT)
                        qv = h < nh ? *reinterpret_cast<const float4*>(qs + (hb + h) * HD + 4 * (j + LPT * c))
                                    : make_float4(0.f, 0.f, 0.f, 0.f);
                    else
                        qv = qf[h][c];
                    s += qv.x * kf[c].x + qv.y * kf[c].y + qv.z * kf[c].z + qv.w * kf[c].w;
                }
                s = group_sum<LPT>(s);
                if (valid && j == 0 && h < nh) sc[h * p.chunk + (tok - ta)] = s * p.scale;
            }
        }
        __syncthreads();

        // ---- per-head max / exp / sum: wave h owns head h ----
        const int len = tb - ta;
        float mx = -1e30f, sum = 0.0f;
        if (wv < nh) {
            float* row = sc + wv * p.chunk;
            for (int i = lane; i < len; i += 64) mx = fmaxf(mx, row[i]);
            mx = wave_max(mx);
            for (int i = lane; i < len; i += 64) {
                const float e = expf(row[i] - mx);
                row[i] = e;
                sum += e;
            }
            sum = wave_sum(sum);
        }
        __syncthreads();

        // ---- pass 2: o = sum_t e_t v_t ----
        if constexpr (SHORT) {
            // V is in LDS: thread (f, tg) sums float4 f of the head block over
            // tokens tg, tg + NTG, ...; the NTG partials meet in LDS
            constexpr int NF = kHeadBlock * HD / 4;
            constexpr int NTG = kThreads / NF;
            const int f = tid % NF, tg = tid / NF;
            const int h = f / (HD / 4), d4 = f % (HD / 4);
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            if (h < nh) {
                const float* prow = sc + h * p.chunk;
                for (int tl = tg; tl < len; tl += NTG) {
                    const float w = prow[tl];
                    const float4 v = *reinterpret_cast<const float4*>(vs + tl * HD + 4 * d4);
                    acc.x += w * v.x;
                    acc.y += w * v.y;
                    acc.z += w * v.z;
                    acc.w += w * v.w;
                }
            }
            float4* r4 = reinterpret_cast<float4*>(red);
            r4[tg * NF + f] = acc;
            if (wv < nh && lane == 0) {
                float* ml = p.part_ml + (static_cast<size_t>(split) * p.n_heads + hk * G + hb + wv) * 2;
                ml[0] = mx;
                ml[1] = sum;
            }
            __syncthreads();
            if (tid < NF && h < nh) {
                float4 t = r4[f];
#pragma unroll
                for (int g = 1; g < NTG; ++g) {
                    const float4 v = r4[g * NF + f];
                    t.x += v.x;
                    t.y += v.y;
                    t.z += v.z;
                    t.w += v.w;
                }
                *reinterpret_cast<float4*>(p.part_o + (static_cast<size_t>(split) * p.n_heads + hk * G + hb + h) * HD +
                                           4 * d4) = t;
            }
            __syncthreads();
            continue;
        }
        float4 of[kHeadBlock][4];
#pragma unroll
        for (int h = 0; h < kHeadBlock; ++h)
#pragma unroll
            for (int c = 0; c < 4; ++c) of[h][c] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int t = ta; t < tb; t += TPP) {
            const int tok = t + ts;
            if (tok < tb) {
                float4 vf[4];
                if (SHORT) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) vf[c] = make_float4(vpre[c].x, vpre[c].y, vpre[c].z, vpre[c].w);
                } else {
                    const float* src = (have_new && tok == p.pos)
                                           ? p.v_new + static_cast<size_t>(hk) * HD
                                           : p.v_cache + static_cast<size_t>(tok) * kv_dim + static_cast<size_t>(hk) * HD;
#pragma unroll
                    for (int c = 0; c < 4; ++c) vf[c] = *reinterpret_cast<const float4*>(src + 4 * (j + LPT * c));
                }
#pragma unroll
                for (int h = 0; h < kHeadBlock; ++h) {
                    const float w = h < nh ? sc[h * p.chunk + (tok - ta)] : 0.0f;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        of[h][c].x += w * vf[c].x;
                        of[h][c].y += w * vf[c].y;
                        of[h][c].z += w * vf[c].z;
                        of[h][c].w += w * vf[c].w;
                    }
                }
            }
        }
        // reduce over the token slots of this wave (lanes with equal j)
#pragma unroll
        for (int h = 0; h < kHeadBlock; ++h)
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int o = LPT; o < 64; o <<= 1) {
                    of[h][c].x += __shfl_xor(of[h][c].x, o, 64);
                    of[h][c].y += __shfl_xor(of[h][c].y, o, 64);
                    of[h][c].z += __shfl_xor(of[h][c].z, o, 64);
                    of[h][c].w += __shfl_xor(of[h][c].w, o, 64);
                }
        if (lane < LPT) {
#pragma unroll
            for (int h = 0; h < kHeadBlock; ++h)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    *reinterpret_cast<float4*>(red + (wv * kHeadBlock + h) * HD + 4 * (j + LPT * c)) = of[h][c];
        }
        // per-head (max, sum) from the owning wave
        if (wv < nh && lane == 0) {
            float* ml = p.part_ml + (static_cast<size_t>(split) * p.n_heads + hk * G + hb + wv) * 2;
            ml[0] = mx;
            ml[1] = sum;
        }
        __syncthreads();
        for (int i = tid; i < nh * HD; i += kThreads) {
            const int h = i / HD, d = i % HD;
            float acc = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) acc += red[(w * kHeadBlock + h) * HD + d];
            p.part_o[(static_cast<size_t>(split) * p.n_heads + hk * G + hb + h) * HD + d] = acc;
        }
        __syncthreads();
    }
}

// Large query-head groups (G = n_heads / n_kv_heads >= 16, head_dim 128),
// e.g. MQA: the G query heads of one KV head are the M dimension of two small
// fp32 matrix products per 64-token sub-chunk, S = Q K^T and O += P V
// (v_mfma_f32_32x32x2f32, fp32 throughout like the reference), so every K/V
// row is read from HBM once.  One work-group (4 waves) owns (KV head, chunk);
// it walks the chunk in sub-chunks with an online softmax (running max and sum
// per head, O rescaled by e^(m_old - m_new)) and leaves the same (o, max, sum)
// partials as attn_chunk_kernel for attn_merge_kernel.
//   S: wave w computes tokens 32 (w % 2) .. + 32 over dims 64 (w / 2) .. + 64;
//      lane l holds Q[l % 32][d] and K[t][d] for the 32 dims d of its half
//      (the order of d inside a dot is free: half g = l / 32 takes dims
//      64 (w / 2) + 32 g .. + 32), the two dim halves meet in LDS.
//   softmax: wave w takes heads 8 w .. 8 w + 7 with lane = token; the eight
//      heads go through each step together (independent DPP max / sum
//      reductions, no LDS round trips), then lane i < 8 updates the running
//      max and sum of head 8 w + i.
//   P V: wave w owns output dims 32 w .. + 32; lane l reads P[l % 32][t] from
//      LDS and V[t][32 w + l % 32] from HBM for tokens t = 32 g + kk.
// MFMA layouts (32x32x2 f32): A[l % 32][l / 32], B[l / 32][l % 32], accumulator
// register r of lane l is D[8 (r / 4) + 4 (l / 32) + r % 4][l % 32].
constexpr int kMqSub = 64;
constexpr int kMqHeads = 32;
constexpr int kMqLd = kMqSub + 4;

__global__ __launch_bounds__(kThreads) void attn_mq_kernel(AttnParams p) {
    constexpr int HD = 128;
    __shared__ __align__(16) float spart[2][kMqHeads][kMqLd];
    __shared__ __align__(16) float pl[kMqHeads][kMqLd];
    __shared__ float alpha_s[kMqHeads], m_s[kMqHeads], l_s[kMqHeads];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int li = lane & 31, g = lane >> 5;
    const int G = p.n_heads / p.n_kv;
    const int hk = blockIdx.x, split = blockIdx.y;
    const int ta = p.t0 + split * p.chunk;
    const int tb = min(p.t1, ta + p.chunk);
    const size_t kv_dim = static_cast<size_t>(p.n_kv) * HD;
    const bool have_new = p.use_new != 0;

    // the work-group whose chunk holds `pos` stores the new K/V row; its own
    // reads of token pos below take k_new / v_new directly
    if (have_new && p.pos >= ta && p.pos < tb) {
        float* kd = p.k_cache + static_cast<size_t>(p.pos) * kv_dim + static_cast<size_t>(hk) * HD;
        float* vd = p.v_cache + static_cast<size_t>(p.pos) * kv_dim + static_cast<size_t>(hk) * HD;
        for (int i = tid; i < HD; i += kThreads) {
            kd[i] = p.k_new[static_cast<size_t>(hk) * HD + i];
            vd[i] = p.v_new[static_cast<size_t>(hk) * HD + i];
        }
    }
    auto krow = [&](int t) -> const float* {
        return (have_new && t == p.pos) ? p.k_new + static_cast<size_t>(hk) * HD
                                        : p.k_cache + static_cast<size_t>(t) * kv_dim + static_cast<size_t>(hk) * HD;
    };
    auto vrow = [&](int t) -> const float* {
        return (have_new && t == p.pos) ? p.v_new + static_cast<size_t>(hk) * HD
                                        : p.v_cache + static_cast<size_t>(t) * kv_dim + static_cast<size_t>(hk) * HD;
    };

    const int tt = wv & 1, dh = wv >> 1;
    const int dq = 64 * dh + 32 * g;  // first dim of this lane's half in the S phase
    float qa[32];
    if (li < G) {
        const float* qr = p.q + (static_cast<size_t>(hk) * G + li) * HD + dq;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float4 v = *reinterpret_cast<const float4*>(qr + 4 * i);
            qa[4 * i] = v.x; qa[4 * i + 1] = v.y; qa[4 * i + 2] = v.z; qa[4 * i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) qa[i] = 0.0f;
    }
    if (tid < kMqHeads) {
        m_s[tid] = -1e30f;
        l_s[tid] = 0.0f;
    }
    floatx16 o;
#pragma unroll
    for (int r = 0; r < 16; ++r) o[r] = 0.0f;
    __syncthreads();

    // Loads run one phase ahead: a sub-chunk's V rows are issued before its
    // S products and the next sub-chunk's K rows right after them, so they
    // arrive while the softmax and P V run.
    float kb[32];
    auto load_k = [&](int sa_) {
        const int tok = sa_ + 32 * tt + li;
        const float* kr = krow(tok < tb ? tok : tb - 1) + dq;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float4 v = *reinterpret_cast<const float4*>(kr + 4 * i);
            kb[4 * i] = v.x; kb[4 * i + 1] = v.y; kb[4 * i + 2] = v.z; kb[4 * i + 3] = v.w;
        }
    };
    if (ta < tb) load_k(ta);
    for (int sa = ta; sa < tb; sa += kMqSub) {
        float vb[32];
#pragma unroll
        for (int kk = 0; kk < 32; ++kk) {
            const int t = sa + 32 * g + kk;
            vb[kk] = vrow(t < tb ? t : tb - 1)[32 * wv + li];
        }
        // ---- S partials over this wave's dim half ----
        {
            floatx16 sacc;
#pragma unroll
            for (int r = 0; r < 16; ++r) sacc[r] = 0.0f;
#pragma unroll
            for (int kk = 0; kk < 32; ++kk) sacc = __builtin_amdgcn_mfma_f32_32x32x2f32(qa[kk], kb[kk], sacc, 0, 0, 0);
            if (sa + kMqSub < tb) load_k(sa + kMqSub);
#pragma unroll
            for (int r = 0; r < 16; ++r) spart[dh][8 * (r >> 2) + 4 * g + (r & 3)][32 * tt + li] = sacc[r];
        }
        __syncthreads();
        // ---- online softmax ----
        {
            const bool valid = sa + lane < tb;
            float sv[8], mo[8], mn[8], su[8];
#pragma unroll
            for (int hh = 0; hh < 8; ++hh) {
                const int h = 8 * wv + hh;
                sv[hh] = valid ? (spart[0][h][lane] + spart[1][h][lane]) * p.scale : -1e30f;
                mo[hh] = m_s[h];
            }
#pragma unroll
            for (int hh = 0; hh < 8; ++hh) mn[hh] = fmaxf(mo[hh], wave_max(sv[hh]));
#pragma unroll
            for (int hh = 0; hh < 8; ++hh) {
                const float e = valid ? expf(sv[hh] - mn[hh]) : 0.0f;
                pl[8 * wv + hh][lane] = e;
                su[hh] = wave_sum(e);
            }
            float m_old = mo[0], m_new = mn[0], sum = su[0];
#pragma unroll
            for (int hh = 1; hh < 8; ++hh) {
                m_old = lane == hh ? mo[hh] : m_old;
                m_new = lane == hh ? mn[hh] : m_new;
                sum = lane == hh ? su[hh] : sum;
            }
            if (lane < 8) {
                const int h = 8 * wv + lane;
                const float a = expf(m_old - m_new);
                alpha_s[h] = a;
                l_s[h] = l_s[h] * a + sum;
                m_s[h] = m_new;
            }
        }
        __syncthreads();
        // ---- O = O e^(m_old - m_new) + P V over this wave's 32 dims ----
        {
#pragma unroll
            for (int r = 0; r < 16; ++r) o[r] *= alpha_s[8 * (r >> 2) + 4 * g + (r & 3)];
            float pa[32];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float4 v = *reinterpret_cast<const float4*>(&pl[li][32 * g + 4 * i]);
                pa[4 * i] = v.x; pa[4 * i + 1] = v.y; pa[4 * i + 2] = v.z; pa[4 * i + 3] = v.w;
            }
#pragma unroll
            for (int kk = 0; kk < 32; ++kk) o = __builtin_amdgcn_mfma_f32_32x32x2f32(pa[kk], vb[kk], o, 0, 0, 0);
        }
        __syncthreads();  // spart / pl / alpha are rewritten by the next sub-chunk
    }
    // partials: unnormalised o, and (max, sum) per head
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int h = 8 * (r >> 2) + 4 * g + (r & 3);
        if (h < G) p.part_o[(static_cast<size_t>(split) * p.n_heads + hk * G + h) * HD + 32 * wv + li] = o[r];
    }
    if (tid < G) {
        float* ml = p.part_ml + (static_cast<size_t>(split) * p.n_heads + hk * G + tid) * 2;
        ml[0] = m_s[tid];
        ml[1] = l_s[tid];
    }
}

// ---------------------------------------------------------------------------
// Causal prefill: B query tokens at positions pos0 .. pos0 + B - 1, each with
// the semantics of one decode step at its position (write its K/V row, then
// attend over its window).  Two launches:
//   attn_prefill_prologue_kernel: the heads-RMSNorm + RoPE prologue of q and
//     k, 16 heads of a token per work-group (the decode prologue's arithmetic,
//     with the token's own host-made cos/sin row), q and k written back, K/V
//     rows stored;
//   attn_prefill_kernel (head_dim 128, G = n_heads / n_kv dividing 32): a
//     work-group owns 128 query rows, 128 / G tokens x the G heads of one KV
//     head, and walks the block's whole key range in 32-key sub-chunks with
//     S^T = K Q^T, online softmax and O += P V (fp16 matrix cores, fp16-pair
//     operands), masking each row to its own causal window, and writes
//     out = O / (l + 1e-12) directly;
//   with a key-split plan a work-group walks one part of a long block's range,
//     and attn_prefill_merge_kernel, a third launch, combines the parts.
struct PrefillParams {
    float* q;             // [B][n_heads * HD], prologue result in place
    float* k;             // [B][n_kv * HD], prologue result in place
    const float* v;       // [B][n_kv * HD]
    float* k_cache;
    float* v_cache;
    float* out;           // [B][n_heads * HD]
    const float* q_gamma;
    const float* k_gamma;
    const float* rope;    // [B][2][HD / 2] cos then sin rows, or null
    int32_t pos0, batch, n_heads, n_kv, sw, norm_qk;
    float scale, eps;
    // key-split plan (null: one work-group per block, longest first):
    // plan[4 y .. 4 y + 3] = (block, slot, first key, last key) of grid row
    // y, slot -1 for a whole block, else the partial slot of that part of a
    // split block, whose (unnormalised o, max, sum) go to part_o / part_ml
    const int32_t* plan;
    float* part_o;   // [slots][n_kv][128 rows][HD]
    float* part_ml;  // [slots][n_kv][128 rows][2]
};

// Work-group (token, kProHeads heads of the token's q heads then KV heads):
// thread (head, d4) holds float4 d4 and d4 + 16 of its head, the RoPE pairs
// of four dims.  The heads' sums of squares are formed 4 lanes per head, as
// head_inv_rms does for one head (the same fp32 lane sums, added in double),
// but for 16 heads at once in one wave: those chains of 32 dependent adds, ten
// heads after one another per wave, were what a token waited for.  KV heads
// also store their K and V rows.  2048 tokens x 40 heads (104 MB): 33 -> 21.0
// us, 300 tokens 18.6 -> 5.7 us.
constexpr int kProHeads = 16;
__global__ __launch_bounds__(kThreads) void attn_prefill_prologue_kernel(PrefillParams p) {
#pragma clang fp contract(off)
    constexpr int HD = 128, LD = HD + 4;  // padded: 16 heads x 4 lanes read distinct banks
    static_assert(kProHeads * HD / 8 == kThreads && kProHeads * 4 == 64, "a pair of float4 per thread, a wave of sums");
    __shared__ __align__(16) float xs[kProHeads * LD];
    __shared__ float inv_s[kProHeads];
    const int t = blockIdx.x, tid = threadIdx.x;
    const int hl = tid / 16, d4 = tid % 16;
    const int head = static_cast<int>(blockIdx.y) * kProHeads + hl, heads = p.n_heads + p.n_kv;
    const bool in = head < heads, is_q = head < p.n_heads;
    const bool rope = p.rope != nullptr, norm = p.norm_qk != 0;
    const int kv = is_q || !in ? 0 : head - p.n_heads;
    const size_t kn = static_cast<size_t>(p.n_kv) * HD;
    float* src = is_q ? p.q + (static_cast<size_t>(t) * p.n_heads + head) * HD
                      : p.k + static_cast<size_t>(t) * kn + static_cast<size_t>(kv) * HD;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a, c = a, s = a, va = a, vb = a;
    float g[8];
    if (in) {
        a = *reinterpret_cast<const float4*>(src + 4 * d4);
        b = *reinterpret_cast<const float4*>(src + 4 * d4 + HD / 2);
        if (!is_q) {
            const float* vr = p.v + static_cast<size_t>(t) * kn + static_cast<size_t>(kv) * HD;
            va = *reinterpret_cast<const float4*>(vr + 4 * d4);
            vb = *reinterpret_cast<const float4*>(vr + 4 * d4 + HD / 2);
        }
        if (rope) {
            const float* rc = p.rope + static_cast<size_t>(t) * HD;
            c = *reinterpret_cast<const float4*>(rc + 4 * d4);
            s = *reinterpret_cast<const float4*>(rc + HD / 2 + 4 * d4);
        }
    }
    const float* gamma = is_q ? p.q_gamma : p.k_gamma;
    if (norm && gamma)
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // (a gamma may be 4-byte aligned only)
            g[e] = gamma[4 * d4 + e];
            g[4 + e] = gamma[HD / 2 + 4 * d4 + e];
        }
    if (norm) {
        *reinterpret_cast<float4*>(&xs[hl * LD + 4 * d4]) = a;
        *reinterpret_cast<float4*>(&xs[hl * LD + 4 * d4 + HD / 2]) = b;
        __syncthreads();
        if (tid < 64) {
            const float* v = &xs[tid / 4 * LD + tid % 4];
            float x[HD / 4];
#pragma unroll
            for (int u = 0; u < HD / 4; ++u) x[u] = v[4 * u];
            float part = 0.0f;
#pragma unroll
            for (int u = 0; u < HD / 4; ++u) part += x[u] * x[u];
            double sum = static_cast<double>(__shfl(part, tid & ~3, 64));
#pragma unroll
            for (int l = 1; l < 4; ++l) sum += static_cast<double>(__shfl(part, (tid & ~3) + l, 64));
            const float mean = static_cast<float>(sum / static_cast<double>(HD));
            if (tid % 4 == 0) inv_s[tid / 4] = 1.0f / sqrtf(mean + p.eps);
        }
        __syncthreads();
    }
    if (!in) return;
    float x1[4] = {a.x, a.y, a.z, a.w}, x2[4] = {b.x, b.y, b.z, b.w};
    if (norm) {
        const float inv = inv_s[hl];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x1[e] = x1[e] * inv;
            x2[e] = x2[e] * inv;
            if (gamma) {
                x1[e] = x1[e] * g[e];
                x2[e] = x2[e] * g[4 + e];
            }
        }
    }
    if (rope) {
        const float cv[4] = {c.x, c.y, c.z, c.w}, sv[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float u = x1[e], w = x2[e];
            x1[e] = u * cv[e] - w * sv[e];
            x2[e] = w * cv[e] + u * sv[e];
        }
    }
    a = make_float4(x1[0], x1[1], x1[2], x1[3]);
    b = make_float4(x2[0], x2[1], x2[2], x2[3]);
    if (norm || rope) {
        *reinterpret_cast<float4*>(src + 4 * d4) = a;
        *reinterpret_cast<float4*>(src + 4 * d4 + HD / 2) = b;
    }
    if (!is_q) {
        const size_t row = static_cast<size_t>(p.pos0 + t) * kn + static_cast<size_t>(kv) * HD;
        *reinterpret_cast<float4*>(p.k_cache + row + 4 * d4) = a;
        *reinterpret_cast<float4*>(p.k_cache + row + 4 * d4 + HD / 2) = b;
        *reinterpret_cast<float4*>(p.v_cache + row + 4 * d4) = va;
        *reinterpret_cast<float4*>(p.v_cache + row + 4 * d4 + HD / 2) = vb;
    }
}

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));

// 8 floats as an fp16 pair: hi = fp16(v), lo = fp16(v - hi) (v - hi is exact
// in fp32), so hi + lo carries about 22 significant bits of v.  Below fp16's
// normal range lo keeps an absolute step of 2^-24, far below what these
// attention sums resolve.
__device__ __forceinline__ void split8(const float (&v)[8], half8_t& hi, half8_t& lo) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const _Float16 h = static_cast<_Float16>(v[i]);
        hi[i] = h;
        lo[i] = static_cast<_Float16>(v[i] - static_cast<float>(h));
    }
}

// The causal batch on the fp16 matrix cores.  A work-group owns 128 query rows
// (128 / G tokens x the G heads of one KV head), a wave 32 of them, and walks
// the rows' key range in 32-key sub-chunks:
//   stage   the sub-chunk's K and V rows are loaded once per work-group (the
//           next sub-chunk's loads are in flight during this one's products),
//           split into fp16 pairs (hi = fp16(v), lo = fp16(v - hi): about 22
//           significant bits) and written to LDS in MFMA operand order;
//   S^T     = K Q^T on v_mfma_f32_32x32x16_f16, three products per K16 slice
//           (hi hi, hi lo, lo hi; the lo lo term is below 2^-22 of the
//           product), Q split once at the start: lane (i, g) ends up holding
//           the scores of query row i (of its wave) for the 16 keys
//           8 a + 4 g + b (a, b = 0..3) of the sub-chunk;
//   softmax the online update of each row's max and sum in registers (the two
//           lane halves of a row meet with one exchange each);
//   O += P V with P straight from those registers as the MFMA's A operand:
//           its K16 slice c holds keys 16 c + 4 g + {0..3, 8..11} in lane half
//           g, and the staged V fragments take the same key order.  O rows
//           are rescaled by the rows' factors through a 32-float LDS array.
// A 64-key sub-chunk of 32 rows with operands from registers and S transposed
// through LDS (the fp32-MFMA form before this) read each K/V row once per 32
// rows instead of once per 128.
// Operands hold |values| < 65504 (fp16's range): q and k after the
// heads-RMSNorm, v and the probabilities in [0, 1].
constexpr int kPfRows = 128;  // query rows (token, head) per work-group
constexpr int kPfKeys = 32;   // keys per sub-chunk

__global__ __launch_bounds__(kThreads, 2) void attn_prefill_kernel(PrefillParams p) {
    constexpr int HD = 128;
    // operand fragments: 8 halves per lane, [slice][lane] for K (A of S^T),
    // [N tile][slice][lane] for V (B of P V)
    __shared__ __align__(16) half8_t khi[HD / 16][64], klo[HD / 16][64];
    __shared__ __align__(16) half8_t vhi[HD / 32][kPfKeys / 16][64], vlo[HD / 32][kPfKeys / 16][64];
    __shared__ __align__(16) float rowf[kWaves][32];  // per-row factors on their way to the O layout
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int li = lane & 31, g = lane >> 5;
    const int G = p.n_heads / p.n_kv, TQ = kPfRows / G;
    const int hk = blockIdx.x;
    int blk = static_cast<int>(gridDim.y) - 1 - static_cast<int>(blockIdx.y);  // longest key ranges first
    int slot = -1;
    if (p.plan) {
        const int4 it = reinterpret_cast<const int4*>(p.plan)[blockIdx.y];
        blk = it.x;
        slot = it.y;
    }
    const int q0 = blk * TQ;
    const int nq = min(TQ, p.batch - q0);
    const int hi_block = p.pos0 + q0 + nq - 1;
    const int lo_block = p.sw > 0 ? max(0, p.pos0 + q0 - p.sw + 1) : 0;
    // this work-group's keys: the block's range, or one part of it
    const int lo_first = p.plan ? reinterpret_cast<const int4*>(p.plan)[blockIdx.y].z : lo_block;
    const int hi_last = p.plan ? reinterpret_cast<const int4*>(p.plan)[blockIdx.y].w : hi_block;
    const size_t kv_dim = static_cast<size_t>(p.n_kv) * HD;
    const size_t q_dim = static_cast<size_t>(p.n_heads) * HD;
    const float* kbase = p.k_cache + static_cast<size_t>(hk) * HD;
    const float* vbase = p.v_cache + static_cast<size_t>(hk) * HD;

    // this lane's query row: row 32 wv + li of the work-group, token
    // (32 wv + li) / G of the block, head (32 wv + li) % G of KV head hk
    const int qrow = 32 * wv + li;
    const int qt = qrow / G;
    const bool qvalid = qt < nq;
    const int q_hi = p.pos0 + q0 + qt;                          // last key of its window
    const int q_lo = p.sw > 0 ? max(0, q_hi - p.sw + 1) : 0;    // first key
    half8_t qh[HD / 16], ql[HD / 16];
    {
        const float* qr = p.q + static_cast<size_t>(q0 + (qvalid ? qt : 0)) * q_dim +
                          (static_cast<size_t>(hk) * G + qrow % G) * HD + 8 * g;
#pragma unroll
        for (int c = 0; c < HD / 16; ++c) {
            const float4 a = *reinterpret_cast<const float4*>(qr + 16 * c);
            const float4 b = *reinterpret_cast<const float4*>(qr + 16 * c + 4);
            float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
            if (!qvalid)
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = 0.0f;
            split8(v, qh[c], ql[c]);
        }
    }

    // staging slots of this thread: K slots tid, tid + 256 (slot s: slice
    // s / 64, lane s % 64 -> key s % 32, dims 16 slice + 8 ((s % 64) / 32));
    // V slots tid, tid + 256 (slot s: N tile s / 128, slice (s / 64) % 2,
    // lane s % 64 -> dim 32 tile + s % 32, keys 16 slice + 4 half + {0..3, 8..11})
    float4 kst[2][2];
    float vst[2][8];
    auto prefetch = [&](int sa) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int sl = tid + 256 * u;
            const int c = sl >> 6, L = sl & 63;
            int key = sa + (L & 31);
            key = key <= hi_last ? key : hi_last;
            const float* kr = kbase + static_cast<size_t>(key) * kv_dim + 16 * c + 8 * (L >> 5);
            kst[u][0] = *reinterpret_cast<const float4*>(kr);
            kst[u][1] = *reinterpret_cast<const float4*>(kr + 4);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int sl = tid + 256 * u;
            const int n = sl >> 7, c = (sl >> 6) & 1, L = sl & 63;
            const int d = 32 * n + (L & 31);
            const int k0 = sa + 16 * c + 4 * (L >> 5);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                int key = k0 + (i & 3) + 8 * (i >> 2);
                key = key <= hi_last ? key : hi_last;
                vst[u][i] = vbase[static_cast<size_t>(key) * kv_dim + d];
            }
        }
    };
    auto stage = [&]() {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int sl = tid + 256 * u;
            const float kv[8] = {kst[u][0].x, kst[u][0].y, kst[u][0].z, kst[u][0].w,
                                 kst[u][1].x, kst[u][1].y, kst[u][1].z, kst[u][1].w};
            half8_t h, l;
            split8(kv, h, l);
            khi[sl >> 6][sl & 63] = h;
            klo[sl >> 6][sl & 63] = l;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int sl = tid + 256 * u;
            half8_t h, l;
            split8(vst[u], h, l);
            vhi[sl >> 7][(sl >> 6) & 1][sl & 63] = h;
            vlo[sl >> 7][(sl >> 6) & 1][sl & 63] = l;
        }
    };

    float m_run = -1e30f, l_run = 0.0f;  // row qrow's running max and sum
    floatx16 o[HD / 32];
#pragma unroll
    for (int n = 0; n < HD / 32; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[n][r] = 0.0f;

    prefetch(lo_first);
    for (int sa = lo_first; sa <= hi_last; sa += kPfKeys) {
        stage();
        __syncthreads();
        if (sa + kPfKeys <= hi_last) prefetch(sa + kPfKeys);
        // S^T for the sub-chunk: rows = keys, columns = this wave's query rows
        floatx16 st;
#pragma unroll
        for (int r = 0; r < 16; ++r) st[r] = 0.0f;
#pragma unroll
        for (int c = 0; c < HD / 16; ++c) {
            const half8_t kh = khi[c][lane], kl = klo[c][lane];
            st = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, qh[c], st, 0, 0, 0);
            st = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, ql[c], st, 0, 0, 0);
            st = __builtin_amdgcn_mfma_f32_32x32x16_f16(kl, qh[c], st, 0, 0, 0);
        }
        // online softmax of row qrow over keys sa + 8 a + 4 g + b (r = 4 a + b),
        // in base 2: scores scaled by scale log2(e), e^(s - m) as one
        // v_exp_f32 of the difference (expf's range reduction took 12% of
        // the kernel; the results move by about 1e-7 relative)
        float mx = -1e30f;
        bool valid[16];
        const float scale2 = p.scale * 1.4426950408889634f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int key = sa + 8 * (r >> 2) + 4 * g + (r & 3);
            valid[r] = qvalid && key >= q_lo && key <= q_hi;
            st[r] = valid[r] ? st[r] * scale2 : -1e30f;
            mx = fmaxf(mx, st[r]);
        }
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float m_new = fmaxf(m_run, mx);
        float e[16], sum = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            e[r] = valid[r] ? __builtin_amdgcn_exp2f(st[r] - m_new) : 0.0f;
            sum += e[r];
        }
        sum += __shfl_xor(sum, 32, 64);
        const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
        l_run = l_run * alpha + sum;
        m_run = m_new;
        // O rows are 8 (r / 4) + 4 g + r % 4 of the wave: their factors via LDS
        if (g == 0) rowf[wv][li] = alpha;
        __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the wave's own writes, read back below
        asm volatile("" ::: "memory");
#pragma unroll
        for (int a4 = 0; a4 < 4; ++a4) {
            const float4 f = *reinterpret_cast<const float4*>(&rowf[wv][8 * a4 + 4 * g]);
#pragma unroll
            for (int n = 0; n < HD / 32; ++n) {
                o[n][4 * a4] *= f.x;
                o[n][4 * a4 + 1] *= f.y;
                o[n][4 * a4 + 2] *= f.z;
                o[n][4 * a4 + 3] *= f.w;
            }
        }
        // O += P V: slice c takes the exponentials e[8 c .. 8 c + 7]
#pragma unroll
        for (int c = 0; c < kPfKeys / 16; ++c) {
            float pv[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) pv[i] = e[8 * c + i];
            half8_t ph, plo;
            split8(pv, ph, plo);
#pragma unroll
            for (int n = 0; n < HD / 32; ++n) {
                const half8_t vh = vhi[n][c][lane], vl = vlo[n][c][lane];
                o[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph, vh, o[n], 0, 0, 0);
                o[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph, vl, o[n], 0, 0, 0);
                o[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(plo, vh, o[n], 0, 0, 0);
            }
        }
        __syncthreads();  // every wave is done with this sub-chunk's K / V fragments
    }
    if (slot >= 0) {
        // a part of a split block: the unnormalised O and the row's (max, sum)
        // for attn_prefill_merge_kernel
        const size_t base = (static_cast<size_t>(slot) * p.n_kv + hk) * kPfRows;
        if (g == 0)
            reinterpret_cast<float2*>(p.part_ml)[base + qrow] = make_float2(m_run, l_run);
#pragma unroll
        for (int a4 = 0; a4 < 4; ++a4)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const int row = 32 * wv + 8 * a4 + 4 * g + b;
#pragma unroll
                for (int n = 0; n < HD / 32; ++n) p.part_o[(base + row) * HD + 32 * n + li] = o[n][4 * a4 + b];
            }
        return;
    }
    // out = O / (l + 1e-12), the rows' sums through LDS like the factors
    if (g == 0) rowf[wv][li] = 1.0f / (l_run + 1e-12f);
    __builtin_amdgcn_s_waitcnt(0xc07f);
    asm volatile("" ::: "memory");
#pragma unroll
    for (int a4 = 0; a4 < 4; ++a4) {
        const float4 f = *reinterpret_cast<const float4*>(&rowf[wv][8 * a4 + 4 * g]);
        const float fr[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int row = 32 * wv + 8 * a4 + 4 * g + b;
            const int t = row / G, h = row % G;
            if (t < nq) {
                float* dst = p.out + static_cast<size_t>(q0 + t) * q_dim + (static_cast<size_t>(hk) * G + h) * HD;
#pragma unroll
                for (int n = 0; n < HD / 32; ++n) dst[32 * n + li] = o[n][4 * a4 + b] * fr[b];
            }
        }
    }
}

// The parts of split block j = blockIdx.y (plan_split[3 j ..]: block, first
// partial slot, parts) for KV head blockIdx.x, a slice of its rows per
// blockIdx.z:
// out = sum_i o_i 2^(m_i - M) / (sum_i l_i 2^(m_i - M) + 1e-12), M = max_i m_i
// (the maxima are in base-2 units, the scores having been scaled by log2 e);
// a part with no key in a row's window has m = -1e30 and weight 0.
constexpr int kPfMaxParts = 8;
__global__ __launch_bounds__(kThreads) void attn_prefill_merge_kernel(PrefillParams p, const int32_t* plan_split) {
    constexpr int HD = 128;
    const int hk = blockIdx.x, j = blockIdx.y;
    const int G = p.n_heads / p.n_kv, TQ = kPfRows / G;
    const int blk = plan_split[3 * j], slot0 = plan_split[3 * j + 1], parts = plan_split[3 * j + 2];
    const int q0 = blk * TQ, nq = min(TQ, p.batch - q0);
    const size_t q_dim = static_cast<size_t>(p.n_heads) * HD;
    // one float4 of one row per thread (grid z: kPfRows HD / 4 / kThreads
    // slices), every part's loads issued together
    {
        const int it = static_cast<int>(blockIdx.z) * kThreads + static_cast<int>(threadIdx.x);
        const int row = it / (HD / 4), d4 = it % (HD / 4);
        const int t = row / G, h = row % G;
        if (t >= nq) return;
        float2 ml[kPfMaxParts];
        float M = -1e30f;
#pragma unroll
        for (int i = 0; i < kPfMaxParts; ++i) {
            if (i < parts) {
                ml[i] = reinterpret_cast<const float2*>(p.part_ml)[(static_cast<size_t>(slot0 + i) * p.n_kv + hk) * kPfRows + row];
                M = fmaxf(M, ml[i].x);
            }
        }
        float l = 0.0f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < kPfMaxParts; ++i) {
            if (i < parts) {
                const float a = __builtin_amdgcn_exp2f(ml[i].x - M);
                const float4 o = reinterpret_cast<const float4*>(
                    p.part_o + ((static_cast<size_t>(slot0 + i) * p.n_kv + hk) * kPfRows + row) * HD)[d4];
                l += ml[i].y * a;
                acc.x += o.x * a;
                acc.y += o.y * a;
                acc.z += o.z * a;
                acc.w += o.w * a;
            }
        }
        const float inv = 1.0f / (l + 1e-12f);
        reinterpret_cast<float4*>(p.out + static_cast<size_t>(q0 + t) * q_dim + (static_cast<size_t>(hk) * G + h) * HD)[d4] =
            make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    }
}

// out[h] = (sum_j o_j e^(m_j - M)) / (sum_j l_j e^(m_j - M) + 1e-12).  Work-
// group (h, y) of a (heads, ny) grid writes float4 columns y nd4 .. + nd4 of
// head h (nd4 = hd / 4 / ny): every work-group forms M and the sum from the
// (max, sum) pairs of all splits and reads only its columns of the partial
// o, so a long window's partials are read by ny times as many CUs.  Thread
// (d4, g) owns column d4 and splits g, g + ng, ...; its first U partial
// loads are issued before the max / sum pass, so the work-group waits on
// memory about once.  U is the smallest of 4, 8, 16 and 32 that covers the
// thread's splits (more loads in flight than needed cost registers and
// occupancy).  The ng per-thread sums of a column meet in an LDS tree.
constexpr int kMergeThreads = 256;
constexpr int kMergeMaxSplit = 4096;
#ifndef GNCX_MERGE_KB
#define GNCX_MERGE_KB 32
#endif
constexpr size_t kMergeBytesPerGroup = static_cast<size_t>(GNCX_MERGE_KB) * 1024;  // partial o per work-group
template <int U>
__global__ __launch_bounds__(kMergeThreads) void attn_merge_kernel(const float* __restrict part_o,
                                                                   const float* __restrict part_ml, int32_t n_split,
                                                                   int32_t n_heads, int32_t hd,
                                                                   float* __restrict out) {
    __shared__ float wgt[kMergeMaxSplit];
    __shared__ float red[2][kMergeThreads / 64];
    __shared__ float4 accs[kMergeThreads];
    const int h = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int nd4 = hd / 4 / static_cast<int>(gridDim.y);  // a power of two from 4 to 64
    const int ng = kMergeThreads / nd4;
    const int d4 = static_cast<int>(blockIdx.y) * nd4 + tid % nd4, g = tid / nd4;
    auto po_at = [&](int s) {
        return *reinterpret_cast<const float4*>(part_o + (static_cast<size_t>(s) * n_heads + h) * hd + 4 * d4);
    };
    // Every load a thread needs is issued here, unconditionally (split
    // indices clamped to the last split, whose weight is then not used), so
    // the kernel waits on memory once: this thread's (max, sum) pair of split
    // tid and its U partial-o float4.
    // (more than kMergeThreads splits: the pairs are read again where used)
    const bool one_ml = n_split <= kMergeThreads;
    auto ml_at = [&](int sp) {
        return *reinterpret_cast<const float2*>(part_ml + (static_cast<size_t>(sp) * n_heads + h) * 2);
    };
    const float2 ml0 = ml_at(tid < n_split ? tid : n_split - 1);
    float4 po[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int sp = g + u * ng;
        po[u] = po_at(sp < n_split ? sp : n_split - 1);
    }
    float m = tid < n_split ? ml0.x : -1e30f;
    if (!one_ml)
        for (int sp = tid + kMergeThreads; sp < n_split; sp += kMergeThreads) m = fmaxf(m, ml_at(sp).x);
    m = wave_max(m);
    if (lane == 0) red[0][wv] = m;
    __syncthreads();
    float M = red[0][0];
    for (int w = 1; w < kMergeThreads / 64; ++w) M = fmaxf(M, red[0][w]);
    float l = 0.0f;
    if (tid < n_split) {
        const float e = expf(ml0.x - M);
        wgt[tid] = e;
        l += ml0.y * e;
    }
    if (!one_ml)
        for (int sp = tid + kMergeThreads; sp < n_split; sp += kMergeThreads) {
            const float2 v = ml_at(sp);
            const float e = expf(v.x - M);
            wgt[sp] = e;
            l += v.y * e;
        }
    l = wave_sum(l);
    if (lane == 0) red[1][wv] = l;
    __syncthreads();
    float lt = 0.0f;
    for (int w = 0; w < kMergeThreads / 64; ++w) lt += red[1][w];
    const float inv = 1.0f / (lt + 1e-12f);
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int sp = g + u * ng;
        const float w = sp < n_split ? wgt[sp] : 0.0f;
        a.x += po[u].x * w;
        a.y += po[u].y * w;
        a.z += po[u].z * w;
        a.w += po[u].w * w;
    }
    for (int sp = g + U * ng; sp < n_split; sp += ng) {
        const float4 v = po_at(sp);
        const float w = wgt[sp];
        a.x += v.x * w;
        a.y += v.y * w;
        a.z += v.z * w;
        a.w += v.w * w;
    }
    accs[tid] = a;
    __syncthreads();
    for (int half = ng / 2; half > 0; half /= 2) {
        if (g < half) {
            const float4 v = accs[tid + half * nd4];
            a.x += v.x;
            a.y += v.y;
            a.z += v.z;
            a.w += v.w;
            accs[tid] = a;
        }
        __syncthreads();
    }
    if (g == 0) {
        float4 r;
        r.x = a.x * inv;
        r.y = a.y * inv;
        r.z = a.z * inv;
        r.w = a.w * inv;
        *reinterpret_cast<float4*>(out + static_cast<size_t>(h) * hd + 4 * d4) = r;
    }
}

hipError_t launch_merge(const float* part_o, const float* part_ml, int32_t n_split, int32_t n_heads, int32_t hd,
                        float* out, hipStream_t stream) {
    // column slices per head: the smallest count that keeps a work-group's
    // share of the partial o within kMergeBytesPerGroup (at least 4 columns each)
    int32_t ny = 1;
    const size_t head_bytes = sizeof(float) * static_cast<size_t>(n_split) * hd;
    while (ny < 16 && hd / 4 / ny > 4 && head_bytes / ny > kMergeBytesPerGroup) ny *= 2;
    const int32_t ng = kMergeThreads / (hd / 4 / ny);  // split groups per column
    const int32_t per = (n_split + ng - 1) / ng;       // splits per thread
    const dim3 grid(n_heads, ny);
    if (per <= 4)
        hipLaunchKernelGGL(attn_merge_kernel<4>, grid, dim3(kMergeThreads), 0, stream, part_o, part_ml, n_split,
                           n_heads, hd, out);
    else if (per <= 8)
        hipLaunchKernelGGL(attn_merge_kernel<8>, grid, dim3(kMergeThreads), 0, stream, part_o, part_ml, n_split,
                           n_heads, hd, out);
    else if (per <= 16)
        hipLaunchKernelGGL(attn_merge_kernel<16>, grid, dim3(kMergeThreads), 0, stream, part_o, part_ml, n_split,
                           n_heads, hd, out);
    else
        hipLaunchKernelGGL(attn_merge_kernel<32>, grid, dim3(kMergeThreads), 0, stream, part_o, part_ml, n_split,
                           n_heads, hd, out);
    return hipGetLastError();
}

struct Plan {
    int32_t t0, t1, chunk, n_split;
};

// LDS per work-group: scores [kHeadBlock][chunk] + wave partials + q + k_new,
// plus the chunk's V rows for a one-pass chunk (kThreads * 16 floats), kept
// within 64 KB by capping the chunk.
constexpr size_t kLdsBudget = 64 * 1024;

size_t lds_base(int32_t chunk, int32_t G, int32_t hd) {
    return sizeof(float) * (static_cast<size_t>(kHeadBlock) * chunk + static_cast<size_t>(kWaves) * kHeadBlock * hd +
                            static_cast<size_t>(G) * hd + hd);
}

// the chunk fits one pass of the work-group and its V rows fit beside the rest
bool one_pass(int32_t chunk, int32_t G, int32_t hd) {
    return chunk <= kThreads / (hd / 16) && lds_base(chunk, G, hd) + sizeof(float) * kThreads * 16 <= kLdsBudget;
}

size_t lds_bytes(int32_t chunk, int32_t G, int32_t hd) {
    return lds_base(chunk, G, hd) + (one_pass(chunk, G, hd) ? sizeof(float) * kThreads * 16 : 0);
}

Plan make_plan(int32_t pos, int32_t sw, int32_t n_kv, int32_t G, int32_t hd) {
    Plan pl;
    pl.t0 = sw > 0 ? (pos - sw + 1 > 0 ? pos - sw + 1 : 0) : 0;
    pl.t1 = pos + 1;
    const int32_t win = pl.t1 - pl.t0;
    auto chunk_for = [&](int32_t groups) {
        int32_t want = groups / (n_kv > 0 ? n_kv : 1);
        if (want < 1) want = 1;
        int32_t c = (win + want - 1) / want;
        c = ((c + 31) / 32) * 32;
        if (c < 32) c = 32;
        return c > kMaxChunk ? kMaxChunk : c;
    };
    int32_t chunk = chunk_for(kTargetGroups);
    if (chunk > 32) chunk = chunk_for(kTargetGroupsLong);
    while (chunk > 32 && lds_bytes(chunk, G, hd) > kLdsBudget) chunk -= 32;
    // the merge weighs at most kMergeMaxSplit chunks
    while ((win + chunk - 1) / chunk > kMergeMaxSplit) chunk += 32;
    pl.chunk = chunk;
    pl.n_split = (win + chunk - 1) / chunk;
    return pl;
}

template <int HD>
hipError_t launch_hd(const AttnArgs& a, const Plan& pl, float* part_o, float* part_ml, hipStream_t stream) {
    AttnParams p{};
    p.q = a.q;
    p.k_new = a.k_new;
    p.v_new = a.v_new;
    p.k_cache = a.k_cache;
    p.v_cache = a.v_cache;
    p.part_o = part_o;
    p.part_ml = part_ml;
    p.q_out = a.q_out;
    p.k_out = a.k_out;
    p.q_gamma = a.q_gamma;
    p.k_gamma = a.k_gamma;
    p.pos = a.pos;
    p.n_heads = a.n_heads;
    p.n_kv = a.n_kv_heads;
    p.t0 = pl.t0;
    p.t1 = pl.t1;
    p.chunk = pl.chunk;
    p.use_new = (a.write_kv && a.k_new && a.v_new) ? 1 : 0;
    p.norm_qk = a.norm_qk;
    p.has_rope = a.rope ? 1 : 0;
    p.scale = a.scale;
    p.eps = a.eps;
    if (a.rope) p.rope = *a.rope;
    else p.rope.half = 0;
    const int G = a.n_heads / a.n_kv_heads;
    const size_t lds = lds_bytes(pl.chunk, G, HD);
    if (lds > kLdsBudget || pl.chunk > kMaxChunk) return hipErrorInvalidValue;  // window too long for one step
    if (one_pass(pl.chunk, G, HD))
        hipLaunchKernelGGL((attn_chunk_kernel<HD, true>), dim3(a.n_kv_heads, pl.n_split), dim3(kThreads), lds, stream,
                           p);
    else
        hipLaunchKernelGGL((attn_chunk_kernel<HD, false>), dim3(a.n_kv_heads, pl.n_split), dim3(kThreads), lds,
                           stream, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    return launch_merge(part_o, part_ml, pl.n_split, a.n_heads, HD, a.out, stream);
}

// Chunks of whole 64-token sub-chunks, about one work-group per CU.
Plan make_mq_plan(int32_t pos, int32_t sw, int32_t n_kv) {
    Plan pl;
    pl.t0 = sw > 0 ? (pos - sw + 1 > 0 ? pos - sw + 1 : 0) : 0;
    pl.t1 = pos + 1;
    const int32_t win = pl.t1 - pl.t0;
    int32_t want = 256 / (n_kv > 0 ? n_kv : 1);
    if (want < 1) want = 1;
    int32_t chunk = (win + want - 1) / want;
    chunk = ((chunk + kMqSub - 1) / kMqSub) * kMqSub;
    while ((win + chunk - 1) / chunk > kMergeMaxSplit) chunk += kMqSub;
    pl.chunk = chunk;
    pl.n_split = (win + chunk - 1) / chunk;
    return pl;
}

hipError_t launch_mq(const AttnArgs& a, const Plan& pl, float* part_o, float* part_ml, hipStream_t stream) {
    AttnParams p{};
    p.q = a.q;
    p.k_new = a.k_new;
    p.v_new = a.v_new;
    p.k_cache = a.k_cache;
    p.v_cache = a.v_cache;
    p.part_o = part_o;
    p.part_ml = part_ml;
    p.pos = a.pos;
    p.n_heads = a.n_heads;
    p.n_kv = a.n_kv_heads;
    p.t0 = pl.t0;
    p.t1 = pl.t1;
    p.chunk = pl.chunk;
    p.use_new = (a.write_kv && a.k_new && a.v_new) ? 1 : 0;
    p.scale = a.scale;
    hipLaunchKernelGGL(attn_mq_kernel, dim3(a.n_kv_heads, pl.n_split), dim3(kThreads), 0, stream, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    return launch_merge(part_o, part_ml, pl.n_split, a.n_heads, 128, a.out, stream);
}

}  // namespace

bool attention_prefill_supported(int32_t n_heads, int32_t n_kv_heads, int32_t head_dim) {
    if (head_dim != 128 || n_kv_heads <= 0 || n_heads <= 0 || n_heads % n_kv_heads != 0) return false;
    const int32_t G = n_heads / n_kv_heads;
    if (G > 32 || 32 % G != 0) return false;
    // up to 128 heads in all.  Nothing in the kernels needs that, but they hold V
    // as fp16 pairs (|v| < 65504) and the per-token steps do not: the route is
    // not widened to shapes that it has not served
    return n_heads + n_kv_heads <= 128;
}

size_t attention_prefill_part_floats(int32_t part_slots, int32_t n_kv_heads) {
    return static_cast<size_t>(part_slots) * n_kv_heads * kPfRows * (128 + 2);
}
constexpr size_t kPfPartMax = size_t{128} << 20;

// The key-split plan of a prefill call.  A block's work is its number of
// 32-key sub-chunks, and two work-groups share a CU, so the kernel's time is
// about the larger of its longest work-group and the total work over the
// resident work-groups.  Blocks longer than a third of the longest (and than 8
// sub-chunks; less where the grid is short, below) are cut into parts of their
// key range of at most that length, each a work-group, whose partial results
// attn_prefill_merge_kernel combines; grid rows are ordered longest first.
// (2048 tokens, 32/8 heads: kernel + merge 200 us per layer unsplit; halves 163
// + 12, thirds best, quarters 149 + 21: the partials' traffic grows with the
// parts.)  Up to 8 sub-chunks in the longest block there is nothing worth a
// second launch: no plan.
// Table: n_items rows of (block, slot, first key, last key), slot -1 for a
// whole block, else its part's index in the partial buffers; then per split
// block (block, first slot, parts).
bool attention_prefill_plan(const PrefillArgs& a, std::vector<int32_t>& tab, int32_t& n_items, int32_t& n_split) {
    n_items = n_split = 0;
    tab.clear();
    if (a.batch <= 0 || a.n_kv_heads <= 0 || a.n_heads % a.n_kv_heads != 0) return false;
    const int32_t G = a.n_heads / a.n_kv_heads, TQ = kPfRows / G;
    const int32_t nblk = (a.batch + TQ - 1) / TQ;
    struct Item {
        int32_t blk, slot, ks, ke;
    };
    std::vector<Item> items;
    std::vector<int32_t> split;
    int32_t maxsub = 0;
    int64_t work = 0;
    auto range = [&](int32_t blk, int32_t& lo, int32_t& hi) {
        const int32_t q0 = blk * TQ, nq = std::min(TQ, a.batch - q0);
        hi = a.pos0 + q0 + nq - 1;
        lo = a.sliding_window > 0 ? std::max(0, a.pos0 + q0 - a.sliding_window + 1) : 0;
    };
    for (int32_t blk = 0; blk < nblk; ++blk) {
        int32_t lo, hi;
        range(blk, lo, hi);
        maxsub = std::max(maxsub, (hi - lo) / kPfKeys + 1);
        work += (hi - lo) / kPfKeys + 1;
    }
    if (maxsub <= 8) return false;
    // few blocks (a short batch, or one on a long cache) leave CUs idle: parts
    // short enough to make 384 work-groups, at least 4 sub-chunks, at most
    // kPfMaxParts of them (whole calls, 32/8 heads, thirds / this: 10 tokens at
    // position 2000 79.5 / 34.3 us, 64 at 1000 54.9 / 26.8, 300 at 0 47.6 /
    // 28.6, the prologue's change included; for 512 work-groups 1000 tokens took
    // 75.7 us against 65.4)
    const int32_t fill = static_cast<int32_t>((work * a.n_kv_heads + 383) / 384);
    const int32_t cut = std::min(std::max<int32_t>(8, (maxsub + 2) / 3),
                                 std::max({4, (maxsub + kPfMaxParts - 1) / kPfMaxParts, fill}));
    int32_t slots = 0;
    for (int32_t blk = nblk - 1; blk >= 0; --blk) {
        int32_t lo, hi;
        range(blk, lo, hi);
        const int32_t nsub = (hi - lo) / kPfKeys + 1;
        if (nsub > cut) {
            const int32_t parts = (nsub + cut - 1) / cut;
            if (parts > kPfMaxParts) return false;
            split.insert(split.end(), {blk, slots, parts});
            for (int32_t q = 0; q < parts; ++q) {
                const int32_t s0 = nsub * q / parts, s1 = nsub * (q + 1) / parts;  // sub-chunks [s0, s1)
                items.push_back({blk, slots + q, lo + kPfKeys * s0, q + 1 == parts ? hi : lo + kPfKeys * s1 - 1});
            }
            slots += parts;
        } else {
            items.push_back({blk, -1, lo, hi});
        }
    }
    // the partial buffers stay within kPfPartMax (a long prompt's plan would
    // need them per 128 rows of every part: it runs unsplit instead)
    if (attention_prefill_part_floats(slots, a.n_kv_heads) * sizeof(float) > kPfPartMax) return false;
    std::stable_sort(items.begin(), items.end(),
                     [](const Item& x, const Item& y) { return x.ke - x.ks > y.ke - y.ks; });
    if (items.size() > 65535 || split.size() / 3 > 65535) return false;
    for (const Item& it : items) tab.insert(tab.end(), {it.blk, it.slot, it.ks, it.ke});
    tab.insert(tab.end(), split.begin(), split.end());
    n_items = static_cast<int32_t>(items.size());
    n_split = static_cast<int32_t>(split.size() / 3);
    return true;
}

// partial slots of a plan: the parts of its split blocks (the last table
// entries: block, first slot, parts)
int32_t attention_prefill_part_slots(const std::vector<int32_t>& tab, int32_t n_items, int32_t n_split) {
    if (n_split <= 0) return 0;
    const size_t last = 4 * static_cast<size_t>(n_items) + 3 * static_cast<size_t>(n_split - 1);
    return tab[last + 1] + tab[last + 2];
}

hipError_t launch_attention_prefill(const PrefillArgs& a, hipStream_t stream) {
    if (a.batch <= 0) return hipSuccess;
    if (!attention_prefill_supported(a.n_heads, a.n_kv_heads, a.head_dim) || a.pos0 < 0) return hipErrorInvalidValue;
    const uintptr_t al = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) |
                         reinterpret_cast<uintptr_t>(a.v) | reinterpret_cast<uintptr_t>(a.out) |
                         reinterpret_cast<uintptr_t>(a.k_cache) | reinterpret_cast<uintptr_t>(a.v_cache);
    if (al & 15u) return hipErrorInvalidValue;
    const int32_t G = a.n_heads / a.n_kv_heads, TQ = kPfRows / G;
    const int32_t nblk = (a.batch + TQ - 1) / TQ;
    if (nblk > 65535) return hipErrorInvalidValue;
    PrefillParams p{};
    p.q = a.q;
    p.k = a.k;
    p.v = a.v;
    p.k_cache = a.k_cache;
    p.v_cache = a.v_cache;
    p.out = a.out;
    p.q_gamma = a.q_gamma;
    p.k_gamma = a.k_gamma;
    p.rope = a.rope;
    p.pos0 = a.pos0;
    p.batch = a.batch;
    p.n_heads = a.n_heads;
    p.n_kv = a.n_kv_heads;
    p.sw = a.sliding_window;
    p.norm_qk = a.norm_qk;
    p.scale = a.scale;
    p.eps = a.eps;
    hipLaunchKernelGGL(attn_prefill_prologue_kernel, dim3(a.batch, (a.n_heads + a.n_kv_heads + kProHeads - 1) / kProHeads),
                       dim3(kThreads), 0, stream, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (!a.plan || a.n_items <= 0) {
        hipLaunchKernelGGL(attn_prefill_kernel, dim3(a.n_kv_heads, nblk), dim3(kThreads), 0, stream, p);
        return hipGetLastError();
    }
    p.plan = a.plan;
    p.part_o = a.part;
    p.part_ml = a.part + static_cast<size_t>(a.part_slots) * a.n_kv_heads * kPfRows * 128;
    hipLaunchKernelGGL(attn_prefill_kernel, dim3(a.n_kv_heads, a.n_items), dim3(kThreads), 0, stream, p);
    e = hipGetLastError();
    if (e != hipSuccess || a.n_split == 0) return e;
    hipLaunchKernelGGL(attn_prefill_merge_kernel, dim3(a.n_kv_heads, a.n_split, kPfRows * 128 / 4 / kThreads),
                       dim3(kThreads), 0, stream, p, a.plan + 4 * a.n_items);
    return hipGetLastError();
}

size_t attention_workspace_bytes(int32_t n_heads, int32_t head_dim, int32_t window) {
    // upper bound over n_kv: chunks of at least 32 tokens, at most kMergeMaxSplit of them
    int32_t n_split = (window + 31) / 32;
    if (n_split > kMergeMaxSplit) n_split = kMergeMaxSplit;
    return sizeof(float) * static_cast<size_t>(n_split) * n_heads * (head_dim + 2) + 256;
}

size_t attention_workspace_need(const AttnArgs& a) {
    if (a.n_heads <= 0 || a.n_kv_heads <= 0 || a.pos < 0 || a.n_heads % a.n_kv_heads != 0) return 0;
    const int32_t G = a.n_heads / a.n_kv_heads;
    const bool mq = a.head_dim == 128 && G >= 16 && G <= kMqHeads && !a.norm_qk && !a.rope;
    const Plan pl = mq ? make_mq_plan(a.pos, a.sliding_window, a.n_kv_heads)
                       : make_plan(a.pos, a.sliding_window, a.n_kv_heads, G, a.head_dim);
    return sizeof(float) * static_cast<size_t>(pl.n_split) * a.n_heads * (a.head_dim + 2);
}

hipError_t launch_attention(const AttnArgs& a, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    if (a.n_heads <= 0 || a.n_kv_heads <= 0 || a.pos < 0) return hipErrorInvalidValue;
    if (a.n_heads % a.n_kv_heads != 0) return hipErrorInvalidValue;
    if (a.rope && a.rope->half * 2 != a.head_dim) return hipErrorInvalidValue;
    const uintptr_t al = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k_cache) |
                         reinterpret_cast<uintptr_t>(a.v_cache) | reinterpret_cast<uintptr_t>(a.out);
    if (al & 15u) return hipErrorInvalidValue;
    const int32_t G = a.n_heads / a.n_kv_heads;
    const bool mq = a.head_dim == 128 && G >= 16 && G <= kMqHeads && !a.norm_qk && !a.rope;
    const Plan pl = mq ? make_mq_plan(a.pos, a.sliding_window, a.n_kv_heads)
                       : make_plan(a.pos, a.sliding_window, a.n_kv_heads, G, a.head_dim);
    const size_t need_o = sizeof(float) * static_cast<size_t>(pl.n_split) * a.n_heads * a.head_dim;
    const size_t need_ml = sizeof(float) * static_cast<size_t>(pl.n_split) * a.n_heads * 2;
    if (need_o + need_ml > workspace_bytes) return hipErrorInvalidValue;
    float* part_o = static_cast<float*>(workspace);
    float* part_ml = reinterpret_cast<float*>(static_cast<char*>(workspace) + need_o);
    if (mq) return launch_mq(a, pl, part_o, part_ml, stream);
    switch (a.head_dim) {
    case 64: return launch_hd<64>(a, pl, part_o, part_ml, stream);
    case 128: return launch_hd<128>(a, pl, part_o, part_ml, stream);
    case 256: return launch_hd<256>(a, pl, part_o, part_ml, stream);
    default: return hipErrorInvalidValue;
    }
}

// ---------------------------------------------------------------------------
// Attention for a tree of drafted tokens over the KV cache.
//
// Several continuations of one sequence, drafted as a tree (speculative
// decoding), are verified in one pass: node i of the tree stands at position
// pos0 + depth(i), and sees the cached rows before pos0 (within its sliding
// window), its ancestors and itself:
//   s_j = scale q_i . k_j,  out_i = sum_j e^(s_j - m) v_j / (sum_j e^(s_j - m) + 1e-12)
// with the decode step's prologue (per-head RMSNorm, NEOX RoPE at the node's
// position) on q and k, and the node's K/V row stored at cache row pos0 + i.
//
// The tree's mask is an interval test.  With the nodes numbered in preorder,
// the subtree of a is the interval [pre_a, end_a), so a is i or an ancestor of
// i exactly when pre_a <= pre_i < end_a, pre_i - pre_a < end_a - pre_a without a
// sign: one compare instead of a T x T mask, and 6 bytes a node, which travel in
// the first launch's arguments.
namespace {

struct TreeParams {
    float* q;
    float* k;
    const float* v;
    float* k_cache;
    float* v_cache;
    float* out;
    const float* q_gamma;
    const float* k_gamma;
    const float* rope;  // [max depth + 1][HD]: cos then sin, or null
    int32_t pos0, n, n_heads, n_kv, sw, norm_qk;
    float scale, eps;
    // the key ranges: first key, keys of one; their parts [range][n_kv][rows_pad]
    int32_t first, chunk, rows_pad;
    float* part_o;    // [..][HD]
    float2* part_ml;  // (max, sum)
    // the tree's table on the device, as the prologue kernel leaves it
    uint32_t* interval;  // [n] pre | end << 16
    uint16_t* depth;     // [n]
    int32_t max_depth;
};

// The decode step's prologue of every node's heads, a wave per head: the
// per-head RMSNorm, then RoPE with the row of the node's depth; KV heads also
// store their cache rows.  The arithmetic is prologue_head_r's of the decode
// step (head_inv_rms, no contraction), so an accepted node's cache row is the
// one that decoding its token would have stored.
// A launch of its own (4 nodes, 40 heads of 128: 3.7 us; 128 nodes, 36 heads: 4.9):
// done by the next kernel's work-groups, its rotations and norms are on the way of
// each of them, 3.7 + 8.3 us against 14.2 (4 nodes at 300).
template <int N>
struct TreeRows {
    uint16_t pre[N], end[N], depth[N];
};
template <int HD, int N>
__global__ __launch_bounds__(kThreads) void tree_prologue_kernel(TreeParams p, TreeRows<N> tree) {
#pragma clang fp contract(off)
    constexpr int H = HD / 2, NR = (H + 63) / 64;
    __shared__ __align__(16) float xs[kWaves][HD];
    const int t = blockIdx.x, lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    // the table travels once, in this launch's arguments, and stays in memory for the
    // next kernel
    if (blockIdx.x == 0 && blockIdx.y == 0)
        for (int i = threadIdx.x; i < p.n; i += kThreads) {
            p.interval[i] = tree.pre[i] | static_cast<uint32_t>(tree.end[i]) << 16;
            p.depth[i] = tree.depth[i];
        }
    const int head = static_cast<int>(blockIdx.y) * kWaves + wv;
    if (head >= p.n_heads + p.n_kv) return;  // whole waves; no barrier below
    const bool is_q = head < p.n_heads;
    const size_t kn = static_cast<size_t>(p.n_kv) * HD;
    const size_t at = static_cast<size_t>(is_q ? 0 : head - p.n_heads) * HD;
    float* src = is_q ? p.q + (static_cast<size_t>(t) * p.n_heads + head) * HD : p.k + t * kn + at;
    const float* gamma = is_q ? p.q_gamma : p.k_gamma;
    float* x = xs[wv];
    for (int i = lane; i < HD; i += 64) x[i] = src[i];
    const float inv = p.norm_qk ? head_inv_rms(x, HD, p.eps, lane) : 1.0f;
    const float* rc = p.rope ? p.rope + static_cast<size_t>(tree.depth[t]) * HD : nullptr;
    const size_t row = (static_cast<size_t>(p.pos0) + t) * kn + at;
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        const int i = lane + 64 * r;
        if (i < H) {
            float a = x[i], b = x[i + H];
            if (p.norm_qk) {
                a = a * inv;
                b = b * inv;
                if (gamma) {
                    a = a * gamma[i];
                    b = b * gamma[i + H];
                }
            }
            if (rc) {
                const float c = rc[i], s = rc[i + H], u = a, w = b;
                a = u * c - w * s;
                b = w * c + u * s;
            }
            if (p.norm_qk || rc) {
                src[i] = a;
                src[i + H] = b;
            }
            if (!is_q) {
                const float* vr = p.v + t * kn + at;
                p.k_cache[row + i] = a;
                p.k_cache[row + i + H] = b;
                p.v_cache[row + i] = vr[i];
                p.v_cache[row + i + H] = vr[i + H];
            }
        }
    }
}

// The products on the fp16 matrix cores.  The kernel below computes, per 32-key
// tile and 32 query rows (node, head) of one KV head,
//   S^T = K Q^T      v_mfma_f32_32x32x16_f16, operands as fp16 pairs, three
//                    products a slice (hi hi, hi lo, lo hi: 2^-22 of the product);
//                    lane (i, g) ends up with query row i's scores of the 16 keys
//                    8 a + 4 g + b
//   O^T += V^T P^T   with P from those registers, and O of row i in lane (i, .):
//                    the softmax factors of a row never cross lanes
// Pairs hold about 22 bits of values from 2^-3 to 2^15, and 2^-25 absolutely
// below.  Every query row, and every group of eight values, is brought there by a
// power of two; a group of eight keys as well unless all of them lie there.  So an
// element keeps 2^-22 of itself or of its row's largest, where that is more.
// The keys' and the row's come back as a factor of the scores.  The values' 2^e
// goes into the weights: those of O are 2^(s + e - max (s + e)), those of the sum
// l 2^(s - max s), two running maxima a row, so that other groups that a row does
// not see have no say in its precision.  Within a group a hidden row may set e, by
// 2^14 above a visible one at most ("odd" keys, below), which leaves the weight of
// the largest term at 2^-2 or more: a pair still holds it to 2^-22, and every smaller
// one to 2^-23 of it.  Value rows of zeros, which any e suits and which bring nothing
// to O, take no part in the second maximum: their weights are added to l alone.
// "Odd" keys, whose key or value row is not finite or lies more than 2^-14 below
// its group's largest, are kept out of the products (0 times an infinity would be
// NaN for the rows that do not see it) and added element by element at the end,
// from lists that the staging leaves (128 nodes at 8192, 32 heads over 4 of 128: 79
// us without odd keys, 109 with one value row in a hundred, 444 with one in eight).
// Parts are left normalised, o_part = sum w v / sum w, with (m, l) beside them:
// no sum of large values can overflow between the kernels.  The reference's
// 1e-12 beside a sum l > 1/2 is below fp32's rounding and left out.
typedef float floatx4 __attribute__((ext_vector_type(4)));

// (by value: a bit cast of a vector's element in place takes the first element)
__device__ __forceinline__ float as_float(uint32_t u) { return __builtin_bit_cast(float, u); }
__device__ __forceinline__ uint32_t as_bits(float f) { return __builtin_bit_cast(uint32_t, f); }
// the float of exponent field `field` (2^(field - 127))
__device__ __forceinline__ float pow2_field(int field) { return __builtin_bit_cast(float, field << 23); }
// amax's exponent field, kept where 2^(+-(14 + e)) are normal floats
__device__ __forceinline__ int scale_field(float amax) {
    const int f = static_cast<int>(as_bits(amax) >> 23) & 0xff;
    return min(max(f, 30), 254);
}
// The exponent field of the power of two that a group of keys of largest element
// top is divided by, `small` if one's largest is below kPlainAbove: 127 (none) for
// larger ones up to 2^14, else one that brings top to 2^14.  A pair's last bit is
// 2^-25 at the least, so either way a key is kept to 2^-22 of its largest element.
constexpr float kPlainAbove = 0.125f;
__device__ __forceinline__ int key_field(float top, bool small) {
    const int f = static_cast<int>(as_bits(top) >> 23) & 0xff;
    return !small && f < 127 + 14 ? 127 : min(max(f, 30), 254) - 14;
}
// max(m, |a|, |b|), NaN if one is
__device__ __forceinline__ float max3_abs(float m, float a, float b) {
    return __builtin_elementwise_maximum(__builtin_elementwise_maximum(m, fabsf(a)), fabsf(b));
}
// max of v and of another lane's `of`, NaN if one is
template <int CTRL>
__device__ __forceinline__ float dpp_maximum(float v, float of) {
    const int o = __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, of), CTRL, 0xf, 0xf, false);
    return __builtin_elementwise_maximum(v, __builtin_bit_cast(float, o));
}
// f of the two halves' values, in every lane
template <class F>
__device__ __forceinline__ float across_halves(float v, F&& f) {
    const auto x = __builtin_amdgcn_permlane32_swap(as_bits(v), as_bits(v), false, false);
    return f(as_float(x[0]), as_float(x[1]));
}
__device__ __forceinline__ float maximum_of(float a, float b) { return __builtin_elementwise_maximum(a, b); }
// the maximum over the wave in every lane, NaN if one is
__device__ __forceinline__ float wave_maximum(float v) {
    v = dpp_maximum<0xb1>(v, v);
    v = dpp_maximum<0x4e>(v, v);
    v = dpp_maximum<0x141>(v, v);
    v = dpp_maximum<0x140>(v, v);
    const auto x = __builtin_amdgcn_permlane16_swap(as_bits(v), as_bits(v), false, false);
    return across_halves(maximum_of(as_float(x[0]), as_float(x[1])), maximum_of);
}

// N floats, times scale, as fp16 pairs: hi nearest, lo nearest to the rest, which
// is exact.  Two values a conversion, and the rest as one mixed fma that reads
// its half of hi in place (written out, as the compiler converts every value once
// more, alone, to subtract it: 2.4 times the issue cycles).
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
template <bool SCALED, int N, class V>
__device__ __forceinline__ void pairs(const float (&v)[N], float scale, V& hi, V& lo) {
    uint32_t h[N / 2], l[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        const float a = v[2 * i], b = v[2 * i + 1];
        h[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(SCALED ? floatx2{a * scale, b * scale} : floatx2{a, b}, half2_t));
        float x, y;
        if constexpr (SCALED) {
            asm("v_fma_mix_f32 %0, %1, %2, -%3 op_sel_hi:[0,0,1]" : "=v"(x) : "v"(a), "v"(scale), "v"(h[i]));
            asm("v_fma_mix_f32 %0, %1, %2, -%3 op_sel:[0,0,1] op_sel_hi:[0,0,1]" : "=v"(y) : "v"(b), "v"(scale), "v"(h[i]));
        } else {
            asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel_hi:[0,0,1]" : "=v"(x) : "v"(a), "v"(h[i]));
            asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel:[0,0,1] op_sel_hi:[0,0,1]" : "=v"(y) : "v"(b), "v"(h[i]));
        }
        l[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(floatx2{x, y}, half2_t));
    }
    hi = __builtin_bit_cast(V, h);
    lo = __builtin_bit_cast(V, l);
}

constexpr int kTreeKeys = 32;        // keys of a tile
constexpr int kTreeMaxChunks = 256;  // key ranges of a call
constexpr float kOddBelow = 1.0f / 16384.0f;

// whether a row of the largest element `row` is odd in a group whose largest
// finite row has `top`
__device__ __forceinline__ bool is_odd(float row, float top) {
    return !(row < __builtin_inff()) || (row > 0.0f && row < top * kOddBelow);
}

// The keys of a range from its first tile with a node on, to the end of its last
// tile, in LDS: a row (pre, lo) sees key t0 + i when pre - first < count (in its
// subtree's interval, first | count << 16; a cached row's is everything, a row's
// behind the range nothing) and, with a window, place >= lo.
struct TreeShared {
    static constexpr int kMost = kMaxTreeNodes + 2 * kTreeKeys;
    __align__(16) uint32_t interval[kMost];
    __align__(16) int32_t place[kMost];  // position
};
__device__ __forceinline__ void load_tree(const TreeParams& p, TreeShared& t, int t0, int c1) {
    for (int i = threadIdx.x; i < (c1 - t0 + kTreeKeys - 1) / kTreeKeys * kTreeKeys; i += kThreads) {
        const int key = t0 + i, node = key - p.pos0;
        uint32_t iv = node < 0 ? 0xffffu << 16 : 0;
        int place = key;
        if (node >= 0 && key < c1) {
            iv = p.interval[node];
            iv -= iv << 16;  // (the end less the first)
            place = p.pos0 + p.depth[node];
        }
        t.interval[i] = iv;
        t.place[i] = place;
    }
}
struct RowPlace {
    uint32_t pre;
    int lo;  // first position of its window
};
__device__ __forceinline__ RowPlace place_of(const TreeParams& p, int node) {
    return {p.interval[node] & 0xffffu, p.sw > 0 ? max(0, p.pos0 + p.depth[node] - p.sw + 1) : 0};
}
__device__ __forceinline__ bool in_interval(uint32_t iv, uint32_t pre) { return pre - (iv & 0xffffu) < iv >> 16; }
// whether a query row sees a key, of the tree's part from t0 on
__device__ __forceinline__ bool sees_key(const TreeShared& t, int t0, const RowPlace& at, int key) {
    return key < t0 ? key >= at.lo : in_interval(t.interval[key - t0], at.pre) && t.place[key - t0] >= at.lo;
}

// One query row a lane: its running maxima of s (m) and of s + e (m + d), and its
// sum.  The maxima are rounded up to whole numbers, so that every factor that brings
// parts to another maximum is a power of two and rounds nothing; the second is kept
// by its distance, as scores of 2^24 and more hold no e.
struct RowState {
    float m, d, l;
};
// The softmax of a tile's scores st, registers 4 h .. of group h with the values'
// exponent ve[h].  Leaves the weights as pairs and returns what O
// so far is to be multiplied with (1: nothing).
__device__ __forceinline__ float tile_softmax(const floatx16& st, const float (&ve)[4], RowState& s, half8_t (&ph)[2],
                                              half8_t (&pl)[2]) {
    float x[4] = {-1e30f, -1e30f, -1e30f, -1e30f};  // (a group without a visible key has no say)
#pragma unroll
    for (int h = 0; h < 4; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[h] = fmaxf(x[h], st[4 * h + i]);
    const auto larger = [](float a, float b) { return fmaxf(a, b); };
    const float m2 = fmaxf(s.m, ceilf(across_halves(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), larger)));
    float mxt = -1e30f;
#pragma unroll
    for (int h = 0; h < 4; ++h) mxt = fmaxf(mxt, x[h] - m2 + ve[h]);
    const float d1 = s.d + (s.m - m2), d2 = fmaxf(d1, ceilf(across_halves(mxt, larger)));
    // 2^(s + e - m - d + 14) = 2^(s - m) 2^(e - d + 14), at most 2^14; the second may
    // pass the largest float where the first is small, so its exponent is added (the
    // bounds are beyond any sum of two: a weight is 0 there either way)
    int f[4];
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int h = 0; h < 4; ++h) f[h] = static_cast<int>(__builtin_amdgcn_fmed3f(ve[h] - d2 + 14.0f, -512.0f, 512.0f));
    half4_t hi[4], lo[4];
#pragma unroll
    for (int a = 0; a < 4; ++a) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            e[i] = __builtin_amdgcn_exp2f(st[4 * a + i] - m2);
            sum[i] += e[i];
            e[i] = __builtin_ldexpf(e[i], f[a]);
        }
        pairs<false>(e, 1.0f, hi[a], lo[a]);
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        ph[c] = __builtin_shufflevector(hi[2 * c], hi[2 * c + 1], 0, 1, 2, 3, 4, 5, 6, 7);
        pl[c] = __builtin_shufflevector(lo[2 * c], lo[2 * c + 1], 0, 1, 2, 3, 4, 5, 6, 7);
    }
    s.l = s.l * __builtin_amdgcn_exp2f(s.m - m2) +
          across_halves((sum[0] + sum[1]) + (sum[2] + sum[3]), [](float a, float b) { return a + b; });
    const float alpha = __builtin_amdgcn_exp2f(d1 - d2);
    s.m = m2;
    s.d = d2;
    return alpha;
}

// Adds the weights of a tile's keys whose value rows are zeros (bits 8 + 4 g .. of
// group h's word) to the sum, and takes them out of the tile (128 nodes at 8192: 79
// us without such rows, 84 with one in a hundred, 100 with one in eight).
typedef uint32_t uint32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void leave_zeros(floatx16& st, const uint32x4& words, int g, RowState& s) {
    float most = -1e30f, sum = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r)
        if (words[r >> 2] >> (8 + 4 * g + (r & 3)) & 1) most = fmaxf(most, st[r]);
    const float m2 = fmaxf(s.m, ceilf(across_halves(most, [](float a, float b) { return fmaxf(a, b); })));
#pragma unroll
    for (int r = 0; r < 16; ++r)
        if (words[r >> 2] >> (8 + 4 * g + (r & 3)) & 1) {
            sum += __builtin_amdgcn_exp2f(st[r] - m2);
            st[r] = -__builtin_inff();
        }
    s.l = s.l * __builtin_amdgcn_exp2f(s.m - m2) + across_halves(sum, [](float a, float b) { return a + b; });
    s.d += s.m - m2;
    s.m = m2;
}

// The odd keys of [t0, t0 + 8) (below c1), by the rule that keeps them out of the
// products, as a mask.
template <int HD>
__device__ uint32_t odd_keys(const float* kbase, const float* vbase, uint32_t kn, int t0, int c1, int lane) {
    // lane = key (eight of them), over its row
    const bool in = lane % 8 + t0 < c1;
    float kmax = 0.0f, vmax = 0.0f;
    const size_t mine = static_cast<size_t>(min(t0 + lane % 8, c1 - 1)) * kn;
#pragma unroll 4
    for (int d = 0; d < HD; d += 4) {
        const floatx4 k = *reinterpret_cast<const floatx4*>(kbase + mine + d), v = *reinterpret_cast<const floatx4*>(vbase + mine + d);
        kmax = max3_abs(max3_abs(kmax, k[0], k[1]), k[2], k[3]);
        vmax = max3_abs(max3_abs(vmax, v[0], v[1]), v[2], v[3]);
    }
    const float ktop = wave_max(in && kmax < __builtin_inff() ? kmax : 0.0f);
    const float vtop = wave_max(in && vmax < __builtin_inff() ? vmax : 0.0f);
    return static_cast<uint32_t>(__ballot(in && lane < 8 && (is_odd(kmax, ktop) || is_odd(vmax, vtop))));
}

// Adds a key to a query row, element by element: to part, its normalised output in
// LDS (float4 d / 4 at 33 (d / 4); the halves of a wave, g, take half of the columns
// each), and to its state.  A weight of 0 takes nothing from a row, whatever it holds.
template <int HD>
__device__ void add_odd_key(const TreeParams& p, const TreeShared& tree, int tree0, const RowPlace& at, float4* part,
                            const float* q, const float* k, const float* v, int key, int g, RowState& s) {
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int d = g * (HD / 2); d < (g + 1) * (HD / 2); d += 4) {
        const floatx4 a = *reinterpret_cast<const floatx4*>(q + d), b = *reinterpret_cast<const floatx4*>(k + d);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] += a[i] * b[i];
    }
    const float x = across_halves((sum[0] + sum[1]) + (sum[2] + sum[3]), [](float a, float b) { return a + b; }) *
                    (p.scale * 1.4426950408889634f);
    if (!sees_key(tree, tree0, at, key) || x == -__builtin_inff()) return;
    const float m2 = fmaxf(s.m, ceilf(x)), a = s.l * __builtin_amdgcn_exp2f(s.m - m2), w = __builtin_amdgcn_exp2f(x - m2);
    s.m = m2;
    s.l = a + w;
    const float fa = a / s.l, fw = w / s.l;
    auto add = [&](float o, float e) { return (fa != 0.0f ? o * fa : 0.0f) + (fw != 0.0f ? fw * e : 0.0f); };
#pragma unroll 4
    for (int d = g * (HD / 8); d < (g + 1) * (HD / 8); ++d) {
        const float4 o = part[33 * d], e = reinterpret_cast<const float4*>(v)[d];
        part[33 * d] = make_float4(add(o.x, e.x), add(o.y, e.y), add(o.z, e.z), add(o.w, e.w));
    }
}

// the wave's normalised part to LDS: float4 column d4 of row li at 33 d4 + li
template <int NN>
__device__ __forceinline__ void store_part(float4* part, const floatx16 (&o)[NN], const RowState& s, int li, int g) {
    const float f = s.l != 0.0f ? 1.0f / s.l : 0.0f;
    // (2^(d - 14) alone may be below the smallest float)
    const int e = static_cast<int>(__builtin_amdgcn_fmed3f(s.d - 14.0f, -512.0f, 512.0f));
    auto out = [&](float x) { return __builtin_ldexpf(x * f, e); };
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int at = 8 * a + 4 * g + b, r = 4 * a + b;  // the lane's column of a column tile
            if constexpr (NN >= 4) {
#pragma unroll
                for (int n = 0; n < NN; n += 4)
                    part[(8 * n + at) * 33 + li] = make_float4(out(o[n][r]), out(o[n + 1][r]), out(o[n + 2][r]), out(o[n + 3][r]));
            } else if (b % 2 == 0) {
                part[at / 2 * 33 + li] = make_float4(out(o[0][r]), out(o[1][r]), out(o[0][r + 1]), out(o[1][r + 1]));
            }
        }
}

// A work-group's rows from the waves' parts in LDS, with (m, l) beside them: to the
// output, or as this key range's part.
template <int HD>
__device__ __forceinline__ void store_rows(const TreeParams& p, const float4* shared, const float2 (*mls)[32], int row0, int hk,
                                           int G, int rows) {
    const bool whole = gridDim.z == 1;
    const size_t prow = (static_cast<size_t>(blockIdx.z) * p.n_kv + hk) * p.rows_pad + row0;
    const int count = min(32 * kWaves, rows - row0) * (HD / 4);
#pragma unroll 4
    for (int i = threadIdx.x; i < count; i += kThreads) {
        const int r = i / (HD / 4), d4 = i % (HD / 4);
        const float2 ml = mls[r / 32][r % 32];
        float4 x = shared[r / 32 * (HD / 4 * 33) + d4 * 33 + r % 32];
        if (whole) {
            const int row = row0 + r;
            if (ml.y != ml.y) x = make_float4(ml.y, ml.y, ml.y, ml.y);  // (an odd key that makes its row NaN)
            reinterpret_cast<float4*>(p.out + (static_cast<size_t>(row / G) * p.n_heads + hk * G + row % G) * HD)[d4] = x;
        } else {
            reinterpret_cast<float4*>(p.part_o + (prow + r) * HD)[d4] = x;
            if (d4 == 0) p.part_ml[prow + r] = ml;
        }
    }
}

// The order of N times (two operand reads from LDS, three products): the reads
// ahead of the products before.  Left alone they come behind those, and are then
// waited for (512 nodes at 32000, 32 heads over 8 of 128: 886 us instead of 861).
template <int N>
__device__ __forceinline__ void interleave_reads() {
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 3, 0);
        if (i + 2 < N) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
}

// A work-group takes 128 query rows of a KV head, 32 a wave, and walks its range
// of keys tile by tile.  Its waves load, scale, split and lay out a tile in LDS as
// operands once for all of them, 8 keys and 8 values each (a group with powers of
// two of its own), two tiles in turn: the next one is laid out, and the one after
// loaded, while this one is in the products, so a tile takes one barrier.  Waves
// without rows (a call of fewer) stage for the others.  Two work-groups a CU fill
// each other's waits.
// Few rows: bound by the reads of the cache (1 node at 32749, 32 heads over 8 of
// 128: 268 MB in a call of 60 us, 4.5 TB/s).  Many: by the matrix cores and the
// work beside them (splitting the tile, the softmax), of which a SIMD has 50 and
// 71 thousand cycles in 136 (128 nodes at 8192, 32 over 4 of 128: 75 us, 0.69
// PFLOP/s of fp16 products; 512 nodes at 32000, 32 over 8: 0.88 to 0.93, a large
// library product of the kind runs at 1.17).
template <int HD, int OCC>
__global__ __launch_bounds__(kThreads, OCC) void tree_rows_kernel(TreeParams p) {
    constexpr int NC = HD / 16, NN = HD / 32;
    constexpr int VW = NN < 4 ? NN : 4;
    constexpr int kPart = HD / 4 * 33;
    constexpr int kTile = NC * 64;  // half8 of a tile's keys' hi (or lo) parts, and of its values'
    constexpr int kShared = kTile * 8 > kPart * kWaves ? kTile * 8 : kPart * kWaves;
    __shared__ __align__(16) float4 shared[kShared];
    __shared__ __align__(16) float kfac[2][kWaves], vexp[2][kWaves];  // [tile in turn][group]: the keys' factor, the values' exponent
    __shared__ __align__(16) uint32_t oddmask[2][kWaves];             // [tile in turn][group]: odd keys | value rows of zeros << 8
    __shared__ float2 mls[kWaves][32];
    // groups with odd keys, by the wave that staged them: tile of the range << 8 |
    // mask; the first tile whose group found no place
    constexpr int kOddGroups = 64;
    __shared__ uint32_t odd_group[kWaves][kOddGroups];
    __shared__ int odd_count[kWaves], odd_more[kWaves];
    __shared__ TreeShared tree;
    half8_t* const khi = reinterpret_cast<half8_t*>(shared);  // [tile in turn][slice][lane]
    half8_t* const klo = khi + 2 * kTile;
    half8_t* const vhi = khi + 4 * kTile;                     // [tile in turn][column tile][slice][lane]
    half8_t* const vlo = khi + 6 * kTile;
    const int tid = threadIdx.x, lane = tid & 63, li = lane & 31, g = lane >> 5;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hk = blockIdx.x, G = p.n_heads / p.n_kv, rows = p.n * G, row0 = static_cast<int>(blockIdx.y) * 32 * kWaves;
    const int c0 = p.first + static_cast<int>(blockIdx.z) * p.chunk, c1 = min(p.pos0 + p.n, c0 + p.chunk);
    const uint32_t kn = static_cast<uint32_t>(p.n_kv) * HD;
    const float* const kbase = p.k_cache + static_cast<size_t>(hk) * HD;
    const float* const vbase = p.v_cache + static_cast<size_t>(hk) * HD;

    // ---- staging: wave w takes keys and values 8 w .. + 8 of a tile: keys eight
    // lanes a row (128 bytes a load), values a lane half a row (register i of half
    // g is row 8 w + 4 g + i)
    auto tile_of = [&](const float* base, int t0) {
        const int n = min(c1 - t0, kTreeKeys);  // none past the range: every load reads zeros
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(base + static_cast<size_t>(t0) * kn), static_cast<short>(0),
                                                 n > 0 ? static_cast<int32_t>((static_cast<uint32_t>(n - 1) * kn + HD) * 4) : 0,
                                                 0x00020000);
    };
    float kst[NN][4], vst[NN][4];
    const int key8 = 8 * wv + lane / 8, part8 = lane % 8;
    const uint32_t kat = (static_cast<uint32_t>(key8) * kn + 4 * part8) * 4;
    const uint32_t vat = ((8 * wv + 4 * g) * kn + VW * li) * 4;
    auto prefetch = [&](int t0) {
        const auto ks = tile_of(kbase, t0), vs = tile_of(vbase, t0);
#pragma unroll
        for (int j = 0; j < NN; ++j) {
            const auto v = __builtin_amdgcn_raw_buffer_load_b128(ks, static_cast<int>(kat + 128 * j), 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) kst[j][i] = as_float(v[i]);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int at = static_cast<int>(vat + static_cast<uint32_t>(r) * kn * 4);
#pragma unroll
            for (int n = 0; n < NN; n += VW) {
                if constexpr (VW == 4) {
                    const auto v = __builtin_amdgcn_raw_buffer_load_b128(vs, at + 128 * n, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; ++i) vst[n + i][r] = as_float(v[i]);
                } else {
                    const auto v = __builtin_amdgcn_raw_buffer_load_b64(vs, at + 128 * n, 0, 0);
#pragma unroll
                    for (int i = 0; i < 2; ++i) vst[n + i][r] = as_float(v[i]);
                }
            }
        }
    };
    auto stage = [&](int b, int t0) {
        uint32_t odd = 0, zeros = 0;  // this group's odd keys, and value rows of zeros beside others
        float krow = 0.0f;
#pragma unroll
        for (int j = 0; j < NN; ++j) krow = max3_abs(max3_abs(krow, kst[j][0], kst[j][1]), kst[j][2], kst[j][3]);
        krow = dpp_maximum<0xb1>(krow, krow);
        krow = dpp_maximum<0x4e>(krow, krow);
        krow = dpp_maximum<0x141>(krow, krow);
        float ktop = wave_maximum(krow);
        if (__ballot(is_odd(krow, ktop))) {
            ktop = wave_max(krow < __builtin_inff() ? krow : 0.0f);
            const uint64_t w = __ballot(is_odd(krow, ktop));
            for (int j = 0; j < 8; ++j) odd |= static_cast<uint32_t>(w >> (8 * j) & 1) << j;
        }
        const int kf = key_field(ktop, __ballot(krow < kPlainAbove) != 0);
        if (kf != 127)
#pragma unroll
            for (int j = 0; j < NN; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) kst[j][i] *= pow2_field(254 - kf);
        // columns 32 j + 4 part8: slice 2 j + part8 / 4, half part8 / 2 % 2, elements 4 (part8 % 2) ..
        const int kslot = (b * kTile + (part8 >> 2) * 64 + (part8 >> 1 & 1) * 32 + key8) * 2 + (part8 & 1);
#pragma unroll
        for (int j = 0; j < NN; ++j) {
            half4_t hi, lo;
            pairs<false>(kst[j], 1.0f, hi, lo);
            reinterpret_cast<half4_t*>(khi)[kslot + 256 * j] = hi;
            reinterpret_cast<half4_t*>(klo)[kslot + 256 * j] = lo;
        }
        float vrow[4], vtop = 0.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            vrow[r] = max3_abs(0.0f, vst[0][r], vst[1][r]);
#pragma unroll
            for (int n = 2; n < NN; n += 2) vrow[r] = max3_abs(vrow[r], vst[n][r], vst[n + 1][r]);
        }
        vtop = wave_maximum(maximum_of(maximum_of(vrow[0], vrow[1]), maximum_of(vrow[2], vrow[3])));
        bool near = vtop < __builtin_inff();
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint64_t here = __ballot(vrow[r] >= vtop * kOddBelow);
            near = near && static_cast<uint32_t>(here) && here >> 32;
        }
        if (!near) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float x = vrow[r];
                x = dpp_maximum<0xb1>(x, x);
                x = dpp_maximum<0x4e>(x, x);
                x = dpp_maximum<0x141>(x, x);
                x = dpp_maximum<0x140>(x, x);
                const auto y = __builtin_amdgcn_permlane16_swap(as_bits(x), as_bits(x), false, false);
                vrow[r] = maximum_of(as_float(y[0]), as_float(y[1]));
            }
            vtop = 0.0f;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (vrow[r] < __builtin_inff()) vtop = fmaxf(vtop, vrow[r]);
            vtop = across_halves(vtop, maximum_of);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const bool bad = is_odd(vrow[r], vtop);
                const uint64_t w = __ballot(bad);
                if (static_cast<uint32_t>(w)) odd |= 1u << r;
                if (w >> 32) odd |= 1u << (r + 4);
                const uint64_t z = __ballot(vrow[r] == 0.0f && vtop > 0.0f);
                if (static_cast<uint32_t>(z)) zeros |= 1u << r;
                if (z >> 32) zeros |= 1u << (r + 4);
#pragma unroll
                for (int n = 0; n < NN; ++n) vst[n][r] = bad ? 0.0f : vst[n][r];
            }
        }
        const int vf = scale_field(vtop) - 14;
        const float vs = pow2_field(254 - vf);
        if (lane == 0) {
            kfac[b][wv] = pow2_field(kf);
            vexp[b][wv] = vtop > 0.0f ? static_cast<float>(vf - 127) : -1e30f;  // (zeros alone: below every other's)
            // (rows past the range are zeros as well, and nobody's)
            oddmask[b][wv] = odd | (zeros & ((1u << min(max(c1 - t0 - 8 * wv, 0), 8)) - 1)) << 8;
            if (odd) {
                const int n = odd_count[wv];
                if (n < kOddGroups) {
                    odd_group[wv][n] = static_cast<uint32_t>(t0 - c0) / kTreeKeys << 8 | odd;
                    odd_count[wv] = n + 1;
                } else {
                    odd_more[wv] = min(odd_more[wv], t0);
                }
            }
        }
        // slice wv / 2, elements 4 (wv % 2) ..
#pragma unroll
        for (int n = 0; n < NN; ++n) {
            half4_t hi, lo;
            pairs<true>(vst[n], vs, hi, lo);
            const int at = (b * kTile + (n * 2 + (wv >> 1)) * 64 + lane) * 2 + (wv & 1);
            reinterpret_cast<half4_t*>(vhi)[at] = hi;
            reinterpret_cast<half4_t*>(vlo)[at] = lo;
        }
    };

    prefetch(c0);
    if (tid < kWaves) {
        odd_count[tid] = 0;
        odd_more[tid] = c1;
    }
    const int tree0 = c0 + max(p.pos0 - c0, 0) / kTreeKeys * kTreeKeys;  // (behind the range: no node in it)
    if (c1 > p.pos0) load_tree(p, tree, tree0, c1);
    // this wave's query rows as operands, in registers
    const int myrow = min(row0 + 32 * wv + li, rows - 1);
    const float* const qrow = p.q + (static_cast<size_t>(myrow / G) * p.n_heads + hk * G + myrow % G) * HD;
    const RowPlace place = place_of(p, myrow / G);
    half8_t qh[NC], ql[NC];
    float qf;
    {
        float x[NC][8], amax = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[c][i] = qrow[16 * c + 8 * g + i];
                amax = fmaxf(amax, fabsf(x[c][i]));
            }
        const int f = scale_field(across_halves(amax, maximum_of));
#pragma unroll
        for (int c = 0; c < NC; ++c) pairs<true>(x[c], pow2_field(254 + 7 - f), qh[c], ql[c]);
        qf = pow2_field(f - 7) * (p.scale * 1.4426950408889634f);
    }
    const int lo_most = p.sw > 0 ? max(0, p.pos0 + p.max_depth - p.sw + 1) : 0;

    // Two work-groups of a CU that start together stay in step, both in the products
    // and both in the softmax; of any 512 that run at a time, the second 256 go first
    // instead (16 heads of 64, 400 rows at 2048 keys: 53.4 -> 50.8 us; 32 over 8 heads
    // of 128, 256 nodes at 4096: 97 -> 89)
    if ((blockIdx.x + gridDim.x * (blockIdx.y + gridDim.y * blockIdx.z)) / 256 & 1) __builtin_amdgcn_s_setprio(1);

    RowState s{-1e30f, 0.0f, 0.0f};
    floatx16 o[NN];
#pragma unroll
    for (int n = 0; n < NN; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[n][r] = 0.0f;

    auto take_tile = [&](int b, int t0) {
        floatx16 st;
#pragma unroll
        for (int r = 0; r < 16; ++r) st[r] = 0.0f;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const half8_t kh = khi[b * kTile + c * 64 + lane], kl = klo[b * kTile + c * 64 + lane];
            st = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, qh[c], st, 0, 0, 0);
            st = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, ql[c], st, 0, 0, 0);
            st = __builtin_amdgcn_mfma_f32_32x32x16_f16(kl, qh[c], st, 0, 0, 0);
        }
        interleave_reads<NC>();
        __builtin_amdgcn_sched_barrier(0);
        const floatx4 kf = *reinterpret_cast<const floatx4*>(kfac[b]), vx = *reinterpret_cast<const floatx4*>(vexp[b]);
        const uint32x4 om = *reinterpret_cast<const uint32x4*>(oddmask[b]);
        const uint32_t apart = __builtin_amdgcn_readfirstlane(om[0] | om[1] | om[2] | om[3]);
        const float ve[4] = {vx[0], vx[1], vx[2], vx[3]}, sf[4] = {kf[0] * qf, kf[1] * qf, kf[2] * qf, kf[3] * qf};
#pragma unroll
        for (int r = 0; r < 16; ++r) st[r] *= sf[r >> 2];
        const float hidden = -__builtin_inff();
        if (t0 + kTreeKeys > p.pos0) {
            typedef int32_t int32x4 __attribute__((ext_vector_type(4)));
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                const int at = t0 - tree0 + 8 * a + 4 * g;
                const uint32x4 iv = *reinterpret_cast<const uint32x4*>(tree.interval + at);
#pragma unroll
                for (int i = 0; i < 4; ++i) st[4 * a + i] = in_interval(iv[i], place.pre) ? st[4 * a + i] : hidden;
                if (p.sw > 0) {
                    const int32x4 x = *reinterpret_cast<const int32x4*>(tree.place + at);
#pragma unroll
                    for (int i = 0; i < 4; ++i) st[4 * a + i] = x[i] >= place.lo ? st[4 * a + i] : hidden;
                }
            }
        } else if (t0 < lo_most) {
#pragma unroll
            for (int r = 0; r < 16; ++r) st[r] = t0 + 8 * (r >> 2) + 4 * g + (r & 3) >= place.lo ? st[r] : hidden;
        }
        if (__builtin_expect(apart != 0, 0)) {
            // by the lane's register: key 8 (r / 4) + 4 g + r % 4
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (om[r >> 2] >> (4 * g + (r & 3)) & 1) st[r] = hidden;
            if (apart >> 8) leave_zeros(st, om, g, s);
        }
        half8_t ph[2], pl[2];
        const float alpha = tile_softmax(st, ve, s, ph, pl);
        if (__ballot(alpha != 1.0f))
#pragma unroll
            for (int n = 0; n < NN; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[n][r] *= alpha;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < NN; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const half8_t vh = vhi[b * kTile + (n * 2 + c) * 64 + lane], vl = vlo[b * kTile + (n * 2 + c) * 64 + lane];
                o[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, ph[c], o[n], 0, 0, 0);
                o[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, pl[c], o[n], 0, 0, 0);
                o[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vl, ph[c], o[n], 0, 0, 0);
            }
        interleave_reads<2 * NN>();
        __builtin_amdgcn_sched_barrier(0);
    };

    __syncthreads();  // no odd keys yet, the tree
    stage(0, c0);
    if (c0 + kTreeKeys < c1) prefetch(c0 + kTreeKeys);
    __syncthreads();
    // (a wave whose 32 rows are none, or see no later node, stages for the others)
    const bool mine = row0 + 32 * wv < rows;
    const int last = mine ? p.pos0 + min(row0 + 32 * wv + 31, rows - 1) / G : -1;
    int b = 0;
    for (int t0 = c0; t0 < c1; t0 += kTreeKeys, b ^= 1) {
        if (t0 + kTreeKeys < c1) stage(b ^ 1, t0 + kTreeKeys);
        if (t0 + 2 * kTreeKeys < c1) prefetch(t0 + 2 * kTreeKeys);
        if (t0 <= last) take_tile(b, t0);
        __syncthreads();  // the next tile is laid out, and this one done with
    }

    float4* const part = shared + wv * kPart;
    store_part<NN>(part, o, s, li, g);
    if (mine && (odd_count[0] | odd_count[1] | odd_count[2] | odd_count[3])) {
        __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the wave's own writes
        asm volatile("" ::: "memory");
        auto add = [&](int t0, uint32_t odd) {
            for (odd = __builtin_amdgcn_readfirstlane(odd); odd; odd &= odd - 1) {
                const int key = t0 + __builtin_ctz(odd);
                const size_t row = static_cast<size_t>(key) * kn;
                add_odd_key<HD>(p, tree, tree0, place, part + li, qrow, kbase + row, vbase + row, key, g, s);
            }
        };
        for (int w = 0; w < kWaves; ++w) {
            for (int i = 0; i < odd_count[w]; ++i)
                add(__builtin_amdgcn_readfirstlane(c0 + static_cast<int>(odd_group[w][i] >> 8) * kTreeKeys + 8 * w),
                    odd_group[w][i] & 0xffu);
            for (int t0 = __builtin_amdgcn_readfirstlane(odd_more[w]); t0 < c1; t0 += kTreeKeys)
                if (t0 + 8 * w < c1) add(t0 + 8 * w, odd_keys<HD>(kbase, vbase, kn, t0 + 8 * w, c1, lane));
        }
    }
    if (g == 0) mls[wv][li] = make_float2(s.m, s.l);
    __syncthreads();
    store_rows<HD>(p, shared, mls, row0, hk, G, rows);
}

// out = sum_c w_c o_c / sum_c w_c with w_c = l_c 2^(m_c - M) over the key
// ranges c.  Bound by the read of the parts: 128 nodes at 8192, 32 heads of 128 (16
// ranges, 34 MB) 11.5 us, 2.9 TB/s; 4 nodes at 300 (10 ranges) 2.7 us.  CG threads share a float4 of the output, each with every CG-th
// range, at most eight, whose loads go out at once; their sums meet in LDS.
constexpr int kTreeMergeLoads = 8;
template <int HD, int CG>
__global__ __launch_bounds__(kThreads) void tree_merge_kernel(TreeParams p, int32_t chunks) {
    static_assert(kTreeMergeLoads * 32 >= kTreeMaxChunks, "32 threads take every range");
    constexpr int kCols = kThreads / CG;  // float4 of a work-group
    __shared__ float4 part[CG][kCols];
    __shared__ float2 mls[CG][kCols];
    const int G = p.n_heads / p.n_kv, rows = p.n * G, hk = blockIdx.y;
    const int col = threadIdx.x % kCols, cg = threadIdx.x / kCols;
    const int i = static_cast<int>(blockIdx.x) * kCols + col, row = min(i / (HD / 4), rows - 1), d4 = i % (HD / 4);
    float2 ml[kTreeMergeLoads];
    float4 v[kTreeMergeLoads];
#pragma unroll
    for (int u = 0; u < kTreeMergeLoads; ++u) {
        const int c = min(cg + u * CG, chunks - 1);
        const size_t at = (static_cast<size_t>(c) * p.n_kv + hk) * p.rows_pad + row;
        ml[u] = p.part_ml[at];
        v[u] = reinterpret_cast<const float4*>(p.part_o + at * HD)[d4];
    }
    // x += f o; a part without a key (f 0) has nothing to add
    auto add = [](float4& x, float f, const float4& o) {
        if (f != 0.0f) {
            x.x += f * o.x;
            x.y += f * o.y;
            x.z += f * o.z;
            x.w += f * o.w;
        }
    };
    // (weights are divided by their sum before they meet the values, whose sum may be
    // past the largest float where their mean is not)
    auto share = [](float L) { return L != 0.0f ? 1.0f / L : 0.0f; };
    float M = -1e30f, L = 0.0f, w[kTreeMergeLoads];
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int u = 0; u < kTreeMergeLoads; ++u) M = fmaxf(M, ml[u].x);
#pragma unroll
    for (int u = 0; u < kTreeMergeLoads; ++u) {
        w[u] = cg + u * CG < chunks ? ml[u].y * __builtin_amdgcn_exp2f(ml[u].x - M) : 0.0f;
        L += w[u];
    }
    float inv = share(L);
#pragma unroll
    for (int u = 0; u < kTreeMergeLoads; ++u) add(x, w[u] * inv, v[u]);
    if constexpr (CG > 1) {
        part[cg][col] = x;
        mls[cg][col] = make_float2(M, L);
        __syncthreads();
        if (cg) return;
        x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        L = 0.0f;
#pragma unroll
        for (int c = 1; c < CG; ++c) M = fmaxf(M, mls[c][col].x);
#pragma unroll
        for (int c = 0; c < CG; ++c) L += mls[c][col].y * __builtin_amdgcn_exp2f(mls[c][col].x - M);
        inv = share(L);
#pragma unroll
        for (int c = 0; c < CG; ++c)
            add(x, mls[c][col].y * __builtin_amdgcn_exp2f(mls[c][col].x - M) * inv, part[c][col]);
    }
    if (i / (HD / 4) >= rows) return;
    reinterpret_cast<float4*>(p.out + (static_cast<size_t>(row / G) * p.n_heads + hk * G + row % G) * HD)[d4] = x;
}

// The split of a call: groups of rows, keys of a range, ranges.
struct TreePlan {
    int32_t groups, first, chunk, chunks, rows_pad;
};

TreePlan tree_plan(const TreeArgs& a) {
    TreePlan pl;
    constexpr int32_t kRows = 32 * kWaves;
    const int32_t rows = a.n * (a.n_heads / a.n_kv_heads);
    pl.groups = (rows + kRows - 1) / kRows;
    pl.rows_pad = pl.groups * kRows;
    pl.first = a.sliding_window > 0 ? std::max(0, a.pos0 - a.sliding_window + 1) : 0;
    const int64_t keys = static_cast<int64_t>(a.pos0) + a.n - pl.first, tiles = (keys + kTreeKeys - 1) / kTreeKeys;
    const int64_t heads = static_cast<int64_t>(pl.groups) * a.n_kv_heads;
    auto ranges_of = [&](int64_t work_groups) {
        return std::min<int64_t>(std::max<int64_t>(1, work_groups / heads), kTreeMaxChunks);
    };
    int64_t ranges = ranges_of(256), per = (tiles + ranges - 1) / ranges;
    // Two work-groups share a CU with heads up to 128.  Twice the ranges halve the
    // tiles of each, and double the parts that meet, the more the more rows there
    // are: worth it from per = ranges on for a group of 128 rows, sooner for fewer.
    // 32 heads over 8 of 128, 256 against 512 work-groups: 128 rows at 2048 (per 3,
    // ranges 32) 27.2 and 30.5 us, at 32000 (32) 95.6 and 88.2; 256 rows at 4096 (9,
    // 16) 38.5 and 41.8, at 8192 (17) 56 and 52; 1024 rows at 300 (5, 4) 48.6 and
    // 44.0; 64 rows at 4096 (5, 32) 26.5 and 27.3, at 8192 (9) 36.0 and 34.3; 16 rows
    // at 2048 (3, 32) 19.1 and 18.3, at 32749 (32) 87 and 60.
    const int64_t used = std::min<int64_t>(kWaves, (rows + 31) / 32);
    if (a.head_dim <= 128 && per * kWaves * kWaves >= ranges * used * used) {
        ranges = ranges_of(512);
        per = (tiles + ranges - 1) / ranges;
    }
    pl.chunk = static_cast<int32_t>(per * kTreeKeys);
    pl.chunks = static_cast<int32_t>((tiles + per - 1) / per);
    return pl;
}

template <int HD, int OCC>
hipError_t launch_tree(const TreeParams& p, const TreeTable& tree, const TreePlan& pl, hipStream_t stream) {
    const int heads = p.n_heads + p.n_kv;
    auto prologue = [&](auto rows) {
        constexpr int N = sizeof(rows) / 6;
        for (int32_t i = 0; i < p.n; ++i) {
            rows.pre[i] = tree.pre[i];
            rows.end[i] = tree.end[i];
            rows.depth[i] = tree.depth[i];
        }
        hipLaunchKernelGGL((tree_prologue_kernel<HD, N>), dim3(p.n, (heads + kWaves - 1) / kWaves), dim3(kThreads), 0, stream, p,
                           rows);
    };
    // (a launch takes the host 1.3 us longer for 3 KB of arguments)
    if (p.n <= 64) prologue(TreeRows<64>{});
    else prologue(TreeRows<kMaxTreeNodes>{});
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((tree_rows_kernel<HD, OCC>), dim3(p.n_kv, pl.groups, pl.chunks), dim3(kThreads), 0, stream, p);
    e = hipGetLastError();
    if (e != hipSuccess || pl.chunks == 1) return e;
    const int64_t n = static_cast<int64_t>(p.n) * (p.n_heads / p.n_kv) * HD / 4;
    auto merge = [&](auto cg) {
        constexpr int CG = decltype(cg)::value, kCols = kThreads / CG;
        hipLaunchKernelGGL((tree_merge_kernel<HD, CG>), dim3(static_cast<uint32_t>((n + kCols - 1) / kCols), p.n_kv),
                           dim3(kThreads), 0, stream, p, pl.chunks);
    };
    if (pl.chunks <= kTreeMergeLoads) merge(std::integral_constant<int, 1>{});
    else if (pl.chunks <= 4 * kTreeMergeLoads) merge(std::integral_constant<int, 4>{});
    else if (pl.chunks <= 8 * kTreeMergeLoads) merge(std::integral_constant<int, 8>{});
    else merge(std::integral_constant<int, 32>{});
    return hipGetLastError();
}

}  // namespace

bool make_tree_table(const int32_t* parents, int32_t n, TreeTable& t) {
    if (n < 1 || n > kMaxTreeNodes) return false;
    int32_t size[kMaxTreeNodes], next[kMaxTreeNodes];  // subtree sizes; the next child's preorder number
    for (int32_t i = 0; i < n; ++i) {
        if (parents[i] < -1 || parents[i] >= i) return false;
        size[i] = 1;
    }
    // a node's number is above its parent's: sizes from the last node up,
    // preorder numbers from the first node down
    for (int32_t i = n - 1; i >= 0; --i)
        if (parents[i] >= 0) size[parents[i]] += size[i];
    int32_t root = 0;
    t.max_depth = 0;
    for (int32_t i = 0; i < n; ++i) {
        const int32_t a = parents[i];
        int32_t& at = a >= 0 ? next[a] : root;
        const int32_t depth = a >= 0 ? t.depth[a] + 1 : 0;
        t.pre[i] = static_cast<uint16_t>(at);
        t.end[i] = static_cast<uint16_t>(at + size[i]);
        t.depth[i] = static_cast<uint16_t>(depth);
        t.max_depth = depth > t.max_depth ? depth : t.max_depth;
        next[i] = at + 1;
        at += size[i];
    }
    return true;
}

namespace {
constexpr size_t kTreeTableBytes = 4096;  // of a workspace: the table, then the parts
static_assert(kMaxTreeNodes * 6 <= kTreeTableBytes);
}  // namespace

size_t attention_tree_workspace_bytes(const TreeArgs& a) {
    const TreePlan pl = tree_plan(a);
    return kTreeTableBytes + (pl.chunks == 1 ? 0 : sizeof(float) * pl.chunks * a.n_kv_heads * pl.rows_pad * (a.head_dim + 2));
}

hipError_t launch_attention_tree(const TreeArgs& a, const TreeTable& tree, void* workspace, size_t workspace_bytes,
                                 hipStream_t stream) {
    if (a.n < 1 || a.n > kMaxTreeNodes || a.pos0 < 0 || a.n_heads < 1 || a.n_kv_heads < 1 ||
        a.n_heads % a.n_kv_heads != 0)
        return hipErrorInvalidValue;
    TreeParams p{};
    p.q = a.q;
    p.k = a.k;
    p.v = a.v;
    p.k_cache = a.k_cache;
    p.v_cache = a.v_cache;
    p.out = a.out;
    p.q_gamma = a.q_gamma;
    p.k_gamma = a.k_gamma;
    p.rope = a.rope;
    p.pos0 = a.pos0;
    p.n = a.n;
    p.n_heads = a.n_heads;
    p.n_kv = a.n_kv_heads;
    p.sw = a.sliding_window;
    p.norm_qk = a.norm_qk;
    p.scale = a.scale;
    p.eps = a.eps;
    p.max_depth = tree.max_depth;
    p.interval = static_cast<uint32_t*>(workspace);
    p.depth = reinterpret_cast<uint16_t*>(p.interval + kMaxTreeNodes);
    const TreePlan pl = tree_plan(a);
    if (workspace_bytes < attention_tree_workspace_bytes(a)) return hipErrorInvalidValue;
    p.first = pl.first;
    p.chunk = pl.chunk;
    p.rows_pad = pl.rows_pad;
    p.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + kTreeTableBytes);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + static_cast<size_t>(pl.chunks) * a.n_kv_heads * pl.rows_pad * a.head_dim);
    switch (a.head_dim) {
    case 64: return launch_tree<64, 2>(p, tree, pl, stream);
    case 128: return launch_tree<128, 2>(p, tree, pl, stream);
    case 256: return launch_tree<256, 1>(p, tree, pl, stream);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace gncx

#include "paged.h"  // many sequences at once
