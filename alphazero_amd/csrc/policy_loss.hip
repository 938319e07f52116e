// policy_loss.hip -- cross entropy of the policy head (PolicyHead's 1x1 convolution and its softmax over all
// c_out * N * N entries, network.hpp:46-65; the policy term of the trainer's loss, train.cpp:90-112) with its gradients,
// without the logits ever being written.
//
//   z[b,o,s]  = sum_c w[o,c] h[b,c,s] + bias[o]                      s = cell of the board, S = N * N
//   lse_b     = log sum over the allowed (o, s) of exp z             loss_b = sum_{t != 0} t (lse_b - z)
//   dz[b,o,s] = r_b (T_b exp(z - lse_b) - t) on allowed entries, 0 elsewhere;  T_b = sum t
//   dh = w^T dz      dw = sum dz h^T      dbias = sum dz
//
// Rows of the work are cells: row r = b * S + s of the flattened batch, 64 rows a step, whatever the board size (a step
// may hold parts of several boards).  az_policy_rows_kernel forms the logits of a step in registers and leaves a row's
// {max, sum of exp, sum t z, sum t}; az_policy_boards_kernel joins a board's rows; az_policy_grad_kernel forms the same
// logits again -- 2 C flop an entry against 8 bytes of a kept fp32 logit written and read -- turns them into dz in LDS
// and multiplies it both ways; az_policy_reduce_kernel adds the workgroups' dw and dbias in a fixed order.
#include "../../include/az_hip.h"
#include "az_learn.h"

#include <cstdarg>
#include <cstdio>

namespace {

int lfail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap; va_start(ap, fmt); vsnprintf(buf, sizeof buf, fmt, ap); va_end(ap);
    return az_internal_fail(code, buf);
}

constexpr int ROWS = 64;                     // rows of a step
constexpr int MAX_GROUPS = 512;              // workgroups of the gradient kernel: two a CU
constexpr float LOG2E = 1.4426950408889634f;

struct PolicyDev {
    const void *h, *w, *bias;
    const float* dense;                      // [B, O * S] or null
    const int *counts, *actions;             // [B], [B, cap]
    const float* probs;                      // [B, cap]
    const unsigned* legal;                   // [B, O * N] or null
    const float* row_scale;                  // [B] or null
    float scale;
    az_f4* rowstat;                          // [B * S] {max, sum, sum t z, sum t}
    az_f4* stats;                            // [B] {lse, T, 1 where a masked action has a target, loss}
    float *loss, *partial;
    void* dh;
    int B, N, S, C, O, cap, nchw;
    int rows, steps;
};

// dynamic LDS of the two product kernels
template <int DT, int OT> struct Lay {
    static constexpr int EP = AzElem<DT>::EP, KS = AzElem<DT>::KS, SZ = 16 / EP;
    static constexpr int OP = (OT * 16 + KS - 1) / KS * KS;          // planes, padded to a step of the contraction over them
    static constexpr int LDT = OT * 16 + 4, LDO = OP + EP;
    static int ldc(int Cp) { return Cp + EP; }                       // 16 bytes of padding: rows start in different banks
    static size_t w_bytes(int Cp) { return (size_t)OP * ldc(Cp) * SZ; }
    static size_t h_bytes(int Cp) { return (size_t)ROWS * ldc(Cp) * SZ; }
    static constexpr size_t z_bytes = (size_t)ROWS * (LDO > LDT ? LDO : LDT) * 4;
};

__device__ __forceinline__ float wave_max(float x) {
    for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o, 64));
    return x;
}
__device__ __forceinline__ float wave_sum(float x) {
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
    return x;
}

// w [O][C] -> LDS [OP][ldc], zero beyond O and C
template <int DT, int OT> __device__ void stage_w(const PolicyDev& a, void* wl, int Cp, int tid, int nt) {
    typedef Lay<DT, OT> L;
    typedef typename AzElem<DT>::T T;
    const int ld = Cp + L::EP;
    for (int i = tid; i < L::OP * ld; i += nt) {
        const int o = i / ld, c = i % ld;
        ((T*)wl)[i] = o < a.O && c < a.C ? ((const T*)a.w)[(size_t)o * a.C + c] : (T)0.f;
    }
}

// The 16-byte pieces of a step's features a thread carries from memory to LDS: rows r0 .., piece p of row r holds
// channels EP * p .. + EP - 1 (zero beyond C and beyond the last row).  Channels last: one load where the piece is whole.
// Channels first: consecutive threads take consecutive cells, EP loads of one element each.
template <int DT, int NP> struct Feat {
    az_i4 v[NP];
    template <int NT> __device__ __forceinline__ void load(const PolicyDev& a, int r0, int pieces, int tid) {
        constexpr int EP = AzElem<DT>::EP;
        typedef typename AzElem<DT>::T T;
        #pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int k = tid + i * NT;
            int row, p;
            if (a.nchw) { row = k % ROWS; p = k / ROWS; } else { row = k / pieces; p = k % pieces; }
            const int r = r0 + row, c0 = p * EP;
            T e[EP];
            #pragma unroll
            for (int j = 0; j < EP; ++j) e[j] = (T)0.f;
            if (row < ROWS && p < pieces && r < a.rows) {
                if (!a.nchw) {
                    const T* src = (const T*)a.h + (size_t)r * a.C + c0;
                    if (c0 + EP <= a.C) {
                        if constexpr (DT == 0) { *(az_f4*)e = *(const az_f4_u*)src; }
                        else { *(az_s8*)e = *(const az_s8_u*)src; }
                    } else {
                        #pragma unroll
                        for (int j = 0; j < EP; ++j) if (c0 + j < a.C) e[j] = src[j];
                    }
                } else {
                    const int b = r / a.S, s = r - b * a.S;
                    const T* src = (const T*)a.h + ((size_t)b * a.C + c0) * a.S + s;
                    #pragma unroll
                    for (int j = 0; j < EP; ++j) if (c0 + j < a.C) e[j] = src[(size_t)j * a.S];
                }
            }
            v[i] = *(az_i4*)e;
        }
    }
    template <int NT> __device__ __forceinline__ void store(const PolicyDev& a, void* hl, int Cp, int pieces, int tid) {
        constexpr int EP = AzElem<DT>::EP, SZ = 16 / EP;
        #pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int k = tid + i * NT;
            int row, p;
            if (a.nchw) { row = k % ROWS; p = k / ROWS; } else { row = k / pieces; p = k % pieces; }
            if (row < ROWS && p < pieces) *(az_i4*)((char*)hl + ((size_t)row * (Cp + EP) + p * EP) * SZ) = v[i];
        }
    }
};

// The sparse targets of a step into t [ROWS][LDT] (zeroed before).  One wave takes a board's entries in their order and
// an LDS add of one wave takes its lanes in theirs, so an action that is named more than once is summed in one order.
// Entries outside 0 .. O * S - 1 are left out.
template <int LDT> __device__ __forceinline__ void scatter_targets(const PolicyDev& a, float* t, int r0, int wave, int waves, int lane) {
    const int last = min(r0 + ROWS, a.rows) - 1;
    const int b0 = r0 / a.S, b1 = last / a.S;
    for (int b = b0 + wave; b <= b1; b += waves) {
        const int n = min(a.counts[b], a.cap);
        const int base = b * a.S - r0;
        for (int e = lane; e < n; e += 64) {
            const int act = a.actions[(size_t)b * a.cap + e];
            if ((unsigned)act >= (unsigned)(a.O * a.S)) continue;
            const int o = act / a.S, idx = base + (act - o * a.S);
            if ((unsigned)idx < (unsigned)ROWS) __hip_atomic_fetch_add(t + idx * LDT + o, a.probs[(size_t)b * a.cap + e], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        }
    }
}

__device__ __forceinline__ bool allowed(const PolicyDev& a, size_t word0, int o, int x) {
    return (a.legal[word0 + (size_t)o * a.N] >> x) & 1u;
}

// Row statistics.  Four waves, 16 rows each, all planes.
template <int DT, int OT, int CB> __global__ void __launch_bounds__(256) az_policy_rows_kernel(PolicyDev a) {
    typedef Lay<DT, OT> L;
    constexpr int NT = 256, NP = CB * 128 / L::EP * ROWS / NT;
    constexpr bool WLDS = !(DT == 0 && CB == 2 && OT >= 6);
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int Cp = (a.C + 31) / 32 * 32, ldc = Cp + L::EP, pieces = Cp / L::EP;
    unsigned char* wl = smem;
    unsigned char* hl = wl + (WLDS ? (size_t)L::OP * ldc * L::SZ : 0);
    float* t = (float*)(hl + (size_t)ROWS * ldc * L::SZ);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, q = lane >> 4;
    if (WLDS) stage_w<DT, OT>(a, wl, Cp, tid, NT);
    const int s_lo = (int)((long long)blockIdx.x * a.steps / gridDim.x), s_hi = (int)((long long)(blockIdx.x + 1) * a.steps / gridDim.x);
    Feat<DT, NP> f;
    if (s_lo < s_hi) f.template load<NT>(a, s_lo * ROWS, pieces, tid);
    for (int st = s_lo; st < s_hi; ++st) {
        const int r0 = st * ROWS;
        __syncthreads();                                             // the step before has read hl and t
        f.template store<NT>(a, hl, Cp, pieces, tid);
        if (a.counts) for (int i = tid; i < ROWS * L::LDT; i += NT) t[i] = 0.f;
        __syncthreads();
        if (st + 1 < s_hi) f.template load<NT>(a, r0 + ROWS, pieces, tid);
        if (a.counts) { scatter_targets<L::LDT>(a, t, r0, wave, 4, lane); __syncthreads(); }
        az_f4 acc[OT];
        #pragma unroll
        for (int ot = 0; ot < OT; ++ot)
            for (int i = 0; i < 4; ++i) { const int o = ot * 16 + q * 4 + i; acc[ot][i] = o < a.O ? az_load<DT>(a.bias, o) : 0.f; }
        for (int k = 0; k < Cp; k += L::KS) {
            const az_i4 hb = az_row_frag<DT>(hl, ldc, wave * 16, k, lane);
            #pragma unroll
            for (int ot = 0; ot < OT; ++ot) {
                az_i4 wa;
                if constexpr (WLDS) wa = az_row_frag<DT>(wl, ldc, ot * 16, k, lane);
                else {
                    const int o = ot * 16 + (lane & 15), c = k + L::EP * q;
                    az_f4 x = {0.f, 0.f, 0.f, 0.f};
                    for (int j = 0; j < 4; ++j) if (o < a.O && c + j < a.C) x[j] = ((const float*)a.w)[(size_t)o * a.C + c + j];
                    wa = __builtin_bit_cast(az_i4, x);
                }
                acc[ot] = az_mma<DT>(wa, hb, acc[ot]);
            }
        }
        const int rl = wave * 16 + (lane & 15), r = r0 + rl;
        if (r < a.rows) {
            const int b = r / a.S, s = r - b * a.S, y = s / a.N, x = s - y * a.N;
            const size_t word0 = (size_t)b * a.O * a.N + y;
            float m = -INFINITY, tz = 0.f, tm = 0.f;
            #pragma unroll
            for (int ot = 0; ot < OT; ++ot) {
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int o = ot * 16 + q * 4 + i;
                    if (o < a.O) {
                        const float tv = a.counts ? t[rl * L::LDT + o] : a.dense[((size_t)b * a.O + o) * a.S + s];
                        if (a.legal && !allowed(a, word0, o, x)) acc[ot][i] = -INFINITY;
                        const float z = acc[ot][i];
                        if (tv != 0.f) { tz += tv * z; tm += tv; }
                        if (!(z <= m)) m = z;                        // (a NaN logit stays in sight: it compares false)
                    } else acc[ot][i] = -INFINITY;
                }
            }
            // four groups of lanes hold a row's planes
            for (int d = 16; d <= 32; d <<= 1) {
                const float om = __shfl_xor(m, d, 64);
                if (!(om <= m)) m = om;
                tz += __shfl_xor(tz, d, 64);
                tm += __shfl_xor(tm, d, 64);
            }
            float l = 0.f;
            if (m != -INFINITY) {
                #pragma unroll
                for (int ot = 0; ot < OT; ++ot)
                    #pragma unroll
                    for (int i = 0; i < 4; ++i) l += __builtin_amdgcn_exp2f((acc[ot][i] - m) * LOG2E);
            }
            for (int d = 16; d <= 32; d <<= 1) l += __shfl_xor(l, d, 64);
            if (q == 0) {
                a.rowstat[r] = az_f4{m, l, tz, tm};
                asm volatile("s_nop 1");                             // (a wide store reads its registers after it has issued)
            }
        }
    }
}

// A board's rows joined: one wave a board.
__global__ void __launch_bounds__(256) az_policy_boards_kernel(PolicyDev a) {
    const int b = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (b >= a.B) return;
    const az_f4* rs = a.rowstat + (size_t)b * a.S;
    float m = -INFINITY, l = 0.f, tz = 0.f, tm = 0.f;
    for (int s = lane; s < a.S; s += 64) {
        const az_f4 v = rs[s];
        tz += v[2];
        tm += v[3];
        if (v[0] == -INFINITY) continue;
        if (v[0] <= m) l += v[1] * __builtin_amdgcn_exp2f((v[0] - m) * LOG2E);
        else { l = (m == -INFINITY ? 0.f : l * __builtin_amdgcn_exp2f((m - v[0]) * LOG2E)) + v[1]; m = v[0]; }
    }
    float M = m;
    for (int d = 32; d > 0; d >>= 1) { const float om = __shfl_xor(M, d, 64); if (!(om <= M)) M = om; }
    l = m == -INFINITY ? 0.f : l * __builtin_amdgcn_exp2f((m - M) * LOG2E);
    l = wave_sum(l);
    tz = wave_sum(tz);
    tm = wave_sum(tm);
    if (lane == 0) {
        const float lse = M == -INFINITY ? -INFINITY : M + logf(l);
        const bool masked = tz == -INFINITY;                         // a target on an action that is not allowed
        const float loss = masked ? INFINITY : (tm != 0.f ? tm * lse : 0.f) - tz;
        a.stats[b] = az_f4{lse, tm, masked ? 1.f : 0.f, loss};
        if (a.loss) a.loss[b] = loss;
    }
}

// Gradients.  Eight waves.  A step: dz of 64 rows (16 rows and half of the planes a wave), then its product with w (16
// rows and half of the channels a wave) and its product with the features (every eighth 16 channels a wave, all planes,
// kept in registers over all of a workgroup's steps).  16-bit features: dz goes to LDS as hi + lo of the type, hi alone
// feeds dh (whose result is rounded to that type anyway), both feed dw (an fp32 sum over all rows: one rounding to 16
// bits of each term would stay in it).
template <int DT, int OT, int CB> __global__ void __launch_bounds__(512) az_policy_grad_kernel(PolicyDev a) {
    typedef Lay<DT, OT> L;
    typedef typename AzElem<DT>::T T;
    constexpr int NT = 512, NP = CB * 128 / L::EP * ROWS / NT, OTH = (OT + 1) / 2;
    constexpr bool WLDS = !(DT == 0 && CB == 2 && OT >= 6);
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int Cp = (a.C + 31) / 32 * 32, ldc = Cp + L::EP, pieces = Cp / L::EP;
    unsigned char* wl = smem;
    unsigned char* hl = wl + (WLDS ? (size_t)L::OP * ldc * L::SZ : 0);
    float* t = (float*)(hl + (size_t)ROWS * ldc * L::SZ);            // the step's targets, then its dz in the same place
    T* zhi = (T*)t;
    T* zlo = zhi + ROWS * L::LDO;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, q = lane >> 4, rt = wave & 3, half = wave >> 2;
    if (WLDS) stage_w<DT, OT>(a, wl, Cp, tid, NT);
    const int s_lo = (int)((long long)blockIdx.x * a.steps / gridDim.x), s_hi = (int)((long long)(blockIdx.x + 1) * a.steps / gridDim.x);
    az_f4 dw[CB][OT];
    #pragma unroll
    for (int i = 0; i < CB; ++i)
        for (int j = 0; j < OT; ++j) dw[i][j] = az_f4{0.f, 0.f, 0.f, 0.f};
    az_f4 db[OTH];
    #pragma unroll
    for (int j = 0; j < OTH; ++j) db[j] = az_f4{0.f, 0.f, 0.f, 0.f};
    Feat<DT, NP> f;
    if (s_lo < s_hi) f.template load<NT>(a, s_lo * ROWS, pieces, tid);
    // fp16: dz is r_b (a mean over the batch: 1 / B) times probabilities that may be 1e-5, below what fp16 resolves.  The
    // workgroup's dz carry a power of two that puts the largest r_b T_b of its boards at 2^9 .. 2^10; it comes off the
    // fp32 sums again.
    float up = 1.f, down = 1.f;
    if constexpr (DT == 1) {
        const int b0 = s_lo * ROWS / a.S, b1 = (min(s_hi * ROWS, a.rows) - 1) / a.S;
        float mx = 0.f;
        for (int b = b0 + tid; b <= b1; b += NT) mx = fmaxf(mx, fabsf(a.scale * (a.row_scale ? a.row_scale[b] : 1.f) * a.stats[b][1]));
        mx = wave_max(mx);
        if (lane == 0) t[wave] = mx;
        __syncthreads();
        for (int w = 0; w < 8; ++w) mx = fmaxf(mx, t[w]);
        if (mx > 0.f && mx < INFINITY) {
            const int e = min(max(10 - (ilogbf(mx) + 1), -100), 100);
            up = ldexpf(1.f, e);
            down = ldexpf(1.f, -e);
        }
    }
    for (int st = s_lo; st < s_hi; ++st) {
        const int r0 = st * ROWS;
        __syncthreads();                                             // the step before has read hl and dz
        f.template store<NT>(a, hl, Cp, pieces, tid);
        if (a.counts) for (int i = tid; i < ROWS * L::LDT; i += NT) t[i] = 0.f;
        __syncthreads();
        if (st + 1 < s_hi) f.template load<NT>(a, r0 + ROWS, pieces, tid);
        const int rl = rt * 16 + (lane & 15), r = r0 + rl;
        const bool live = r < a.rows;
        const int b = live ? r / a.S : 0, s = live ? r - b * a.S : 0, y = s / a.N, x = s - y * a.N;
        az_f4 tv[OTH];
        if (a.counts) {
            scatter_targets<L::LDT>(a, t, r0, wave, 8, lane);
            __syncthreads();
            #pragma unroll
            for (int j = 0; j < OTH; ++j) {
                const int ot = half * OTH + j;
                tv[j] = ot < OT ? *(const az_f4*)(t + rl * L::LDT + ot * 16 + q * 4) : az_f4{0.f, 0.f, 0.f, 0.f};
            }
            __syncthreads();                                         // dz takes the targets' place
        } else {
            #pragma unroll
            for (int j = 0; j < OTH; ++j)
                for (int i = 0; i < 4; ++i) {
                    const int o = (half * OTH + j) * 16 + q * 4 + i;
                    tv[j][i] = live && o < a.O ? a.dense[((size_t)b * a.O + o) * a.S + s] : 0.f;
                }
        }
        az_f4 acc[OTH];
        #pragma unroll
        for (int j = 0; j < OTH; ++j)
            for (int i = 0; i < 4; ++i) { const int o = (half * OTH + j) * 16 + q * 4 + i; acc[j][i] = o < a.O ? az_load<DT>(a.bias, o) : 0.f; }
        for (int k = 0; k < Cp; k += L::KS) {
            const az_i4 hb = az_row_frag<DT>(hl, ldc, rt * 16, k, lane);
            #pragma unroll
            for (int j = 0; j < OTH; ++j) {
                const int ot = half * OTH + j;
                if (ot >= OT) continue;
                az_i4 wa;
                if constexpr (WLDS) wa = az_row_frag<DT>(wl, ldc, ot * 16, k, lane);
                else {
                    const int o = ot * 16 + (lane & 15), c = k + L::EP * q;
                    az_f4 v = {0.f, 0.f, 0.f, 0.f};
                    for (int e = 0; e < 4; ++e) if (o < a.O && c + e < a.C) v[e] = ((const float*)a.w)[(size_t)o * a.C + c + e];
                    wa = __builtin_bit_cast(az_i4, v);
                }
                acc[j] = az_mma<DT>(wa, hb, acc[j]);
            }
        }
        const az_f4 bst = live ? a.stats[b] : az_f4{0.f, 0.f, 0.f, 0.f};
        const float rs = live ? up * (a.scale * (a.row_scale ? a.row_scale[b] : 1.f)) : 0.f;
        const float rT = rs * bst[1];
        const size_t word0 = (size_t)b * a.O * a.N + y;
        // one plane and no target outside the allowed actions: the bias moves every logit alike, its gradient is zero
        const bool bias_counts = a.O > 1 || bst[2] != 0.f;
        #pragma unroll
        for (int j = 0; j < OTH; ++j) {
            const int ot = half * OTH + j;
            if (ot * 16 >= L::OP) continue;
            az_f4 dz;
            #pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int o = ot * 16 + q * 4 + i;
                const bool on = live && o < a.O && !(a.legal && !allowed(a, word0, o, x));
                dz[i] = on ? rT * __builtin_amdgcn_exp2f((acc[j][i] - bst[0]) * LOG2E) - rs * tv[j][i] : 0.f;
                if (bias_counts) db[j][i] += dz[i];
            }
            if constexpr (DT == 0) *(az_f4*)((float*)zhi + rl * L::LDO + ot * 16 + q * 4) = dz;
            else {
                az_s4 hi, lo;
                #pragma unroll
                for (int i = 0; i < 4; ++i) { hi[i] = az_to16<DT>(dz[i]); lo[i] = az_to16<DT>(dz[i] - az_from16<DT>(hi[i])); }
                *(az_s4*)((short*)zhi + rl * L::LDO + ot * 16 + q * 4) = hi;
                *(az_s4*)((short*)zlo + rl * L::LDO + ot * 16 + q * 4) = lo;
            }
        }
        __syncthreads();
        // dh: rows of the tile are channels, columns are cells
        for (int ct = half; ct * 16 < Cp; ct += 2) {
            az_f4 d = {0.f, 0.f, 0.f, 0.f};
            #pragma unroll
            for (int k = 0; k < L::OP; k += L::KS) {
                az_i4 wa;
                if constexpr (WLDS) wa = az_col_frag<DT>(wl, ldc, k, ct * 16, lane);
                else {
                    const int c = ct * 16 + (lane & 15);
                    az_f4 v = {0.f, 0.f, 0.f, 0.f};
                    for (int e = 0; e < 4; ++e) { const int o = k + 4 * q + e; if (o < a.O && c < a.C) v[e] = ((const float*)a.w)[(size_t)o * a.C + c]; }
                    wa = __builtin_bit_cast(az_i4, v);
                }
                d = az_mma<DT>(wa, az_row_frag<DT>(zhi, L::LDO, rt * 16, k, lane), d);
            }
            if constexpr (DT == 1) d *= down;
            const int c = ct * 16 + q * 4;
            if (live && c < a.C) {
                if (!a.nchw) {
                    const size_t at = (size_t)r * a.C + c;
                    if (c + 4 <= a.C) {
                        if constexpr (DT == 0) *(az_f4_u*)((float*)a.dh + at) = d;
                        else *(az_s4_u*)((short*)a.dh + at) = az_s4{az_to16<DT>(d[0]), az_to16<DT>(d[1]), az_to16<DT>(d[2]), az_to16<DT>(d[3])};
                    } else for (int i = 0; i < 4; ++i) if (c + i < a.C) az_store<DT>(a.dh, at + i, d[i]);
                } else for (int i = 0; i < 4; ++i) if (c + i < a.C) az_store<DT>(a.dh, ((size_t)b * a.C + c + i) * a.S + s, d[i]);
            }
        }
        // dw: rows of the tile are planes, columns are channels, the contraction runs over the step's rows
        #pragma unroll
        for (int ci = 0; ci < CB; ++ci) {
            const int ct = wave + 8 * ci;
            if (ct * 16 >= Cp) continue;
            #pragma unroll
            for (int k = 0; k < ROWS; k += L::KS) {
                const az_i4 hb = az_col_frag<DT>(hl, ldc, k, ct * 16, lane);
                #pragma unroll
                for (int ot = 0; ot < OT; ++ot) {
                    dw[ci][ot] = az_mma<DT>(az_col_frag<DT>(zhi, L::LDO, k, ot * 16, lane), hb, dw[ci][ot]);
                    if constexpr (DT != 0) dw[ci][ot] = az_mma<DT>(az_col_frag<DT>(zlo, L::LDO, k, ot * 16, lane), hb, dw[ci][ot]);
                }
            }
        }
    }
    float* out = a.partial + (size_t)blockIdx.x * ((size_t)a.O * a.C + a.O);
    #pragma unroll
    for (int ci = 0; ci < CB; ++ci) {
        const int c = (wave + 8 * ci) * 16 + (lane & 15);
        #pragma unroll
        for (int ot = 0; ot < OT; ++ot)
            for (int i = 0; i < 4; ++i) {
                const int o = ot * 16 + q * 4 + i;
                if (o < a.O && c < a.C) out[(size_t)o * a.C + c] = dw[ci][ot][i] * down;
            }
    }
    __syncthreads();
    float* red = t;                                                  // [4][OT * 16]
    #pragma unroll
    for (int j = 0; j < OTH; ++j) {
        const int ot = half * OTH + j;
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            float v = db[j][i];
            for (int d = 1; d < 16; d <<= 1) v += __shfl_xor(v, d, 64);
            if (ot < OT && (lane & 15) == 0) red[rt * OT * 16 + ot * 16 + q * 4 + i] = v;
        }
    }
    __syncthreads();
    for (int o = tid; o < a.O; o += NT) out[(size_t)a.O * a.C + o] = ((red[o] + red[OT * 16 + o]) + (red[2 * OT * 16 + o] + red[3 * OT * 16 + o])) * down;
}

// Workgroups' sums added in their order: 64 entries a block, 8 slices of the workgroups.
__global__ void __launch_bounds__(512) az_policy_reduce_kernel(const float* partial, int groups, int O, int C, float* dw, float* dbias) {
    __shared__ float red[8][64];
    const int n = O * C + O, i = blockIdx.x * 64 + (threadIdx.x & 63), slice = threadIdx.x >> 6;
    const int lo = slice * groups / 8, hi = (slice + 1) * groups / 8;
    float v = 0.f;
    if (i < n) {
        #pragma unroll 8
        for (int g = lo; g < hi; ++g) v += partial[(size_t)g * n + i];
    }
    red[slice][threadIdx.x & 63] = v;
    __syncthreads();
    if (slice == 0 && i < n) {
        for (int k = 1; k < 8; ++k) v += red[k][threadIdx.x];
        if (i < O * C) dw[i] = v; else dbias[i - O * C] = v;
    }
}

template <int DT, int OT, int CB> hipError_t launch_products(const PolicyDev& a, bool grad, int groups, hipStream_t stream) {
    typedef Lay<DT, OT> L;
    const int Cp = (a.C + 31) / 32 * 32;
    const bool wlds = !(DT == 0 && CB == 2 && OT >= 6);
    const size_t lds = (wlds ? L::w_bytes(Cp) : 0) + L::h_bytes(Cp) + L::z_bytes;
    const void* fn = grad ? (const void*)az_policy_grad_kernel<DT, OT, CB> : (const void*)az_policy_rows_kernel<DT, OT, CB>;
    if (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    if (grad) az_policy_grad_kernel<DT, OT, CB><<<groups, 512, lds, stream>>>(a);
    else az_policy_rows_kernel<DT, OT, CB><<<groups, 256, lds, stream>>>(a);
    return hipGetLastError();
}
template <int DT, int OT> hipError_t launch_c(const PolicyDev& a, bool grad, int groups, hipStream_t stream) {
    return a.C <= 128 ? launch_products<DT, OT, 1>(a, grad, groups, stream) : launch_products<DT, OT, 2>(a, grad, groups, stream);
}
template <int DT> hipError_t launch_o(const PolicyDev& a, bool grad, int groups, hipStream_t stream) {
    if (a.O <= 16) return launch_c<DT, 1>(a, grad, groups, stream);
    if (a.O <= 32) return launch_c<DT, 2>(a, grad, groups, stream);
    if (a.O <= 64) return launch_c<DT, 4>(a, grad, groups, stream);
    if (a.O <= 96) return launch_c<DT, 6>(a, grad, groups, stream);
    return launch_c<DT, 8>(a, grad, groups, stream);
}
hipError_t launch_dt(int dtype, const PolicyDev& a, bool grad, int groups, hipStream_t stream) {
    if (dtype == AZ_F32) return launch_o<0>(a, grad, groups, stream);
    if (dtype == AZ_F16) return launch_o<1>(a, grad, groups, stream);
    return launch_o<2>(a, grad, groups, stream);
}

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

int groups_of(long long steps) { return (int)(steps < MAX_GROUPS ? steps : MAX_GROUPS); }

// shape and range checks that need no pointer; 0 or the recorded error
int check_shape(const az_policy_loss_args* p) {
    if (!p) return lfail(AZ_E_ARG, "null argument: args");
    if (p->B < 0) return lfail(AZ_E_ARG, "batch %d is negative", p->B);
    if (p->N < 1 || p->N > 32) return lfail(AZ_E_ARG, "board side %d unsupported (1..32)", p->N);
    if (p->C < 1 || p->C > 256) return lfail(AZ_E_ARG, "%d channels unsupported (1..256)", p->C);
    if (p->c_out < 1 || p->c_out > 128) return lfail(AZ_E_ARG, "%d policy channels unsupported (1..128)", p->c_out);
    if (p->dtype != AZ_F32 && p->dtype != AZ_F16 && p->dtype != AZ_BF16) return lfail(AZ_E_ARG, "element type %d unknown (AZ_F32, AZ_F16, AZ_BF16)", p->dtype);
    if (p->layout != AZ_CHANNELS_FIRST && p->layout != AZ_CHANNELS_LAST) return lfail(AZ_E_ARG, "layout %d unknown (AZ_CHANNELS_FIRST, AZ_CHANNELS_LAST)", p->layout);
    if ((long long)p->B * p->N * p->N > 0x7fffff00ll) return lfail(AZ_E_ARG, "batch %d of %dx%d boards has too many cells for one call", p->B, p->N, p->N);
    return AZ_OK;
}

}  // namespace

extern "C" size_t az_policy_loss_workspace(const az_policy_loss_args* p) {
    if (check_shape(p) != AZ_OK) return 0;
    const size_t rows = (size_t)p->B * p->N * p->N;
    size_t n = up256(rows * sizeof(az_f4)) + up256((size_t)p->B * sizeof(az_f4));
    if (p->d_weight) n += up256((size_t)groups_of((long long)(rows + ROWS - 1) / ROWS) * ((size_t)p->c_out * p->C + p->c_out) * 4);
    return n ? n : 256;
}

extern "C" int az_policy_loss_dev(const az_policy_loss_args* p, void* workspace, size_t workspace_bytes, void* stream) {
    const int rc = check_shape(p);
    if (rc != AZ_OK) return rc;
    const bool grad = p->d_features || p->d_weight || p->d_bias;
    if (grad && !((p->d_features || p->B == 0) && p->d_weight && p->d_bias)) return lfail(AZ_E_ARG, "null argument: the gradients come together (d_features, d_weight, d_bias)");
    if (!grad && !p->loss && !p->stats && p->B > 0) return lfail(AZ_E_ARG, "null argument: nothing to compute (loss, stats and gradients are null)");
    if (p->stats_given && (!p->stats || !grad)) return lfail(AZ_E_ARG, "stats_given needs stats and the gradients");
    if (p->B > 0) {
        if (!p->features) return lfail(AZ_E_ARG, "null argument: features");
        if (!p->weight) return lfail(AZ_E_ARG, "null argument: weight");
        if (!p->bias) return lfail(AZ_E_ARG, "null argument: bias");
        if (!p->target && !p->counts) return lfail(AZ_E_ARG, "null argument: target or counts / actions / probs");
        if (p->target && p->counts) return lfail(AZ_E_ARG, "targets are dense (target) or sparse (counts), not both");
        if (p->counts && (p->cap < 0 || (p->cap > 0 && (!p->actions || !p->probs)))) return lfail(AZ_E_ARG, "null argument: actions / probs (cap %d)", p->cap);
        const size_t esz = p->dtype == AZ_F32 ? 4 : 2;
        if (((size_t)p->features | (size_t)p->weight | (size_t)p->bias | (size_t)p->d_features) % esz) return lfail(AZ_E_ARG, "a tensor is not aligned to its element type");
        if (((size_t)p->target | (size_t)p->counts | (size_t)p->actions | (size_t)p->probs | (size_t)p->legal | (size_t)p->row_scale | (size_t)p->loss |
             (size_t)p->d_weight | (size_t)p->d_bias) % 4) return lfail(AZ_E_ARG, "a tensor is not aligned to its element type");
    }
    if ((size_t)p->stats % 16) return lfail(AZ_E_ARG, "stats needs 16-byte alignment");
    const size_t need = az_policy_loss_workspace(p);
    if (!workspace) return lfail(AZ_E_ARG, "null argument: workspace");
    if ((size_t)workspace % 256) return lfail(AZ_E_ARG, "workspace needs 256-byte alignment");
    if (workspace_bytes < need) return lfail(AZ_E_CAPACITY, "workspace has %zu bytes, az_policy_loss_workspace asks for %zu", workspace_bytes, need);
    AzDeviceGuard dev(p->device);
    if (!dev.ok) return lfail(AZ_E_HIP, "device %d cannot be used (no HIP device: libazhip has no CPU fallback)", p->device);
    hipStream_t st = (hipStream_t)stream;
    PolicyDev a = {};
    a.h = p->features; a.w = p->weight; a.bias = p->bias; a.dense = p->target; a.counts = p->counts; a.actions = p->actions; a.probs = p->probs;
    a.legal = p->legal; a.row_scale = p->row_scale; a.scale = p->scale; a.loss = p->loss; a.dh = p->d_features;
    a.B = p->B; a.N = p->N; a.S = p->N * p->N; a.C = p->C; a.O = p->c_out; a.cap = p->cap; a.nchw = p->layout == AZ_CHANNELS_FIRST;
    a.rows = a.B * a.S; a.steps = (a.rows + ROWS - 1) / ROWS;
    unsigned char* ws = (unsigned char*)workspace;
    a.rowstat = (az_f4*)ws; ws += up256((size_t)a.rows * sizeof(az_f4));
    a.stats = p->stats ? (az_f4*)p->stats : (az_f4*)ws; ws += up256((size_t)a.B * sizeof(az_f4));
    a.partial = (float*)ws;
    const int groups = groups_of(a.steps);
    hipError_t e = hipSuccess;
    if (a.B > 0 && !p->stats_given) {
        e = launch_dt(p->dtype, a, false, groups, st);
        if (e == hipSuccess) { az_policy_boards_kernel<<<(a.B + 3) / 4, 256, 0, st>>>(a); e = hipGetLastError(); }
    }
    if (e == hipSuccess && grad) {
        if (a.B > 0) e = launch_dt(p->dtype, a, true, groups, st);
        if (e == hipSuccess) {
            az_policy_reduce_kernel<<<(a.O * a.C + a.O + 63) / 64, 512, 0, st>>>(a.partial, a.B > 0 ? groups : 0, a.O, a.C, p->d_weight, p->d_bias);
            e = hipGetLastError();
        }
    }
    if (e != hipSuccess) return lfail(AZ_E_HIP, "az_policy_loss_dev: launch failed: %s", hipGetErrorString(e));
    return AZ_OK;
}
