// policy_loss.hip -- cross entropy of the policy head (PolicyHead's 1x1 convolution and its softmax over all
// c_out * N * N entries, network.hpp:46-65; the policy term of the trainer's loss, train.cpp:90-112) with its gradients,
// without the logits ever being written.
//
//   z[b,o,s]  = sum_c w[o,c] h[b,c,s] + bias[o]                      s = cell of the board, S = N * N
//   lse_b     = log sum over the allowed (o, s) of exp z             loss_b = sum_{t != 0} t (lse_b - z)
//   dz[b,o,s] = r_b (T_b exp(z - lse_b) - t) on allowed entries, 0 elsewhere;  T_b = sum t
//   dh = w^T dz      dw = sum dz h^T      dbias = sum dz
//
// Rows of the work are cells: row r = b * S + s of the flattened batch.  A step is up to 64 rows: a block of one board, or
// several whole boards where they are small (32 cells or fewer).  az_policy_rows_kernel forms the logits of a step in registers and leaves a row's
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
constexpr size_t LDS_BYTES = 160 * 1024;
constexpr int MAX_GROUPS = 512;              // workgroups of the gradient kernel: two a CU
constexpr int ENTRIES = 1024;                // sparse targets of a step's boards kept in LDS; longer lists are read from memory
constexpr int MAX_BOARDS = 16;               // boards of a step
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
    const float *wpad, *wpadt;               // fp32 weights that do not fit LDS: padded copies
    void* dh;
    int B, N, S, C, O, cap, nchw;
    int rows, steps;                         // steps = work items of up to 64 rows
    int nb, blocks;                          // boards a step holds (blocks = 1), or blocks a board is cut into (nb = 1)
};

// dynamic LDS of the two product kernels
template <int DT, int OT> struct Lay {
    static constexpr int EP = AzElem<DT>::EP, KS = AzElem<DT>::KS, SZ = 16 / EP;
    static constexpr int OP = (OT * 16 + KS - 1) / KS * KS;          // planes, padded to a step of the contraction over them
    static constexpr int LDT = OT * 16 + 4, LDO = OP + EP;
    __host__ __device__ static int ldc(int Cp) { return Cp + EP; }                       // 16 bytes of padding: rows start in different banks
    __host__ __device__ static size_t w_bytes(int Cp) { return (size_t)OP * ldc(Cp) * SZ; }
    __host__ __device__ static size_t h_bytes(int Cp) { return (size_t)ROWS * ldc(Cp) * SZ; }
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

// A step: rows rbase .. rbase + n - 1 of the flattened batch, cells cell0 .. of board b0 (or whole boards b0 ..).
struct Step { int b0, cell0, rbase, n; };
__device__ __forceinline__ Step step_at(const PolicyDev& a, int it) {
    Step s;
    if (a.nb > 1) {
        s.b0 = it * a.nb; s.cell0 = 0; s.rbase = s.b0 * a.S;
        s.n = min(a.nb, a.B - s.b0) * a.S;
    } else {
        s.b0 = it / a.blocks; s.cell0 = (it - s.b0 * a.blocks) * ROWS; s.rbase = s.b0 * a.S + s.cell0;
        s.n = min(ROWS, a.S - s.cell0);
    }
    return s;
}

// The 16-byte pieces of a step's features a thread carries from memory to LDS: rows r0 .., piece p of row r holds
// channels EP * p .. + EP - 1 (zero beyond C and beyond the last row).  Channels last: one load where the piece is whole.
// Channels first: consecutive threads take consecutive cells, EP loads of one element each.
template <int DT, int NP> struct Feat {
    az_i4 v[NP];
    template <int NT> __device__ __forceinline__ void load(const PolicyDev& a, const Step& st, int pieces, int tid) {
        constexpr int EP = AzElem<DT>::EP;
        typedef typename AzElem<DT>::T T;
        #pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int k = tid + i * NT;
            int row, p;
            if (a.nchw) { row = k % ROWS; p = k / ROWS; } else { row = k / pieces; p = k % pieces; }
            const int r = st.rbase + row, c0 = p * EP;
            T e[EP];
            #pragma unroll
            for (int j = 0; j < EP; ++j) e[j] = (T)0.f;
            if (row < st.n && p < pieces) {
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

// What a step's boards need beside the features, brought to LDS when the board changes: the legal-move words, and the
// sparse targets as {row of the step's boards * 256 + plane, value} (entries that are left out: -1).
struct BoardLds {
    unsigned* words;
    int planes;                                                      // words of a line: the planes, padded to 16
    int* key;
    float* val;
    bool listed;                                                     // the entries fit
};
__host__ __device__ inline int entry_room(int nb, int cap) { return (long long)nb * cap <= ENTRIES ? nb * cap : 0; }
__device__ __forceinline__ int entry_key(const PolicyDev& a, int act, int bb) {
    if ((unsigned)act >= (unsigned)(a.O * a.S)) return -1;
    const int o = act / a.S;
    return (bb * a.S + act - o * a.S) * 256 + o;
}
__device__ __forceinline__ int entry_at(const PolicyDev& a, const Step& st, int e, float& v) {
    const int bb = a.nb > 1 ? e / a.cap : 0, k = e - bb * a.cap;
    const size_t at = (size_t)(st.b0 + bb) * a.cap + k;
    if (k >= a.counts[st.b0 + bb]) return -1;
    v = a.probs[at];
    return entry_key(a, a.actions[at], bb);
}
__device__ __forceinline__ void stage_boards(const PolicyDev& a, const BoardLds& l, int b0, int tid, int nt) {
    const int boards = min(a.nb, a.B - b0);
    if (a.legal)                                                     // [board, plane, row] -> [board, row][plane]: a lane reads its row's words four at a time
        for (int i = tid; i < boards * a.O * a.N; i += nt) {
            const int bo = i / a.N, y = i - bo * a.N, bb = a.nb > 1 ? bo / a.O : 0;
            l.words[(bb * a.N + y) * l.planes + bo - bb * a.O] = a.legal[(size_t)b0 * a.O * a.N + i];
        }
    if (a.counts && l.listed)
        for (int e = tid; e < boards * a.cap; e += nt) {
            const int bb = a.nb > 1 ? e / a.cap : 0, k = e - bb * a.cap;
            const size_t at = (size_t)(b0 + bb) * a.cap + k;
            const bool live = k < a.counts[b0 + bb];
            l.key[e] = live ? entry_key(a, a.actions[at], bb) : -1;
            l.val[e] = live ? a.probs[at] : 0.f;
        }
}
// The sparse targets of a step into t [ROWS][LDT] (zeroed before).  A wave adds the entries of its own planes in their
// order (an LDS add takes a wave's lanes in theirs), so an action that is named more than once is summed in one order.
template <int LDT, int WAVES> __device__ __forceinline__ void scatter_targets(const PolicyDev& a, const BoardLds& l, float* t, const Step& st, int wave, int lane) {
    const int boards = min(a.nb, a.B - st.b0), n = boards * a.cap;
    for (int e = lane; e < n; e += 64) {
        int key;
        float v = 0.f;
        if (l.listed) { key = l.key[e]; v = l.val[e]; }
        else key = entry_at(a, st, e, v);
        const int o = key & 255, row = (key >> 8) - st.cell0;
        if (key >= 0 && o % WAVES == wave && (unsigned)row < (unsigned)ROWS)
            __hip_atomic_fetch_add(t + row * LDT + o, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
}

// fp32 weights of more than 32 planes and 128 channels do not fit LDS beside a step: a zero-padded copy [OP][Cp] and one
// transposed [Cp][OP] lie in the workspace, and fragments come from the caches (the fp32 matrix instructions take 32
// cycles for the 512 bytes of operands that a wave loads).
__global__ void __launch_bounds__(256) az_policy_pad_weight_kernel(const float* w, float* pad, float* padt, int O, int C, int OP, int Cp) {
    for (int i = blockIdx.x * 256 + threadIdx.x; i < OP * Cp; i += gridDim.x * 256) {
        const int o = i / Cp, c = i % Cp;
        const float v = o < O && c < C ? w[(size_t)o * C + c] : 0.f;
        pad[i] = v;
        padt[c * OP + o] = v;
    }
}
template <int DT, int OT, int CB> __host__ __device__ constexpr bool w_in_lds() { return !(DT == 0 && CB == 2 && OT >= 4); }

// LDS of the product kernels, in this order; zb: bytes of the kernel's own tile (logits or dz)
template <int DT, int OT, int CB, bool HBUF> struct Smem {
    typedef Lay<DT, OT> L;
    unsigned char *w, *h;
    float *t, *bias;
    BoardLds b;
    __device__ __forceinline__ Smem(unsigned char* p, const PolicyDev& a, int Cp, size_t zb) {
        w = p; p += w_in_lds<DT, OT, CB>() ? L::w_bytes(Cp) : 0;
        h = p; p += HBUF ? L::h_bytes(Cp) : 0;
        t = (float*)p; p += zb;
        bias = (float*)p; p += OT * 16 * 4;
        b.words = (unsigned*)p; p += a.legal ? (size_t)a.nb * a.N * OT * 16 * 4 : 0;
        b.planes = OT * 16;
        const int room = a.counts ? entry_room(a.nb, a.cap) : 0;
        b.listed = room > 0;
        b.key = (int*)p; p += (size_t)room * 4;
        b.val = (float*)p;
    }
    static size_t bytes(const PolicyDev& a, int Cp, size_t zb) {
        return (w_in_lds<DT, OT, CB>() ? L::w_bytes(Cp) : 0) + (HBUF ? L::h_bytes(Cp) : 0) + zb + OT * 16 * 4 + (a.counts ? (size_t)entry_room(a.nb, a.cap) * 8 : 0) +
               (a.legal ? (size_t)a.nb * a.N * OT * 16 * 4 : 0);
    }
};

// Fragments of 16 rows of the features straight from memory: row r of the batch (this lane's, live or not), all channels.
template <int DT, int KT> struct RowFrags {
    az_i4 v[KT];
    __device__ __forceinline__ void load(const PolicyDev& a, const Step& st, int rl, int q) {
        constexpr int EP = AzElem<DT>::EP, KS = AzElem<DT>::KS;
        typedef typename AzElem<DT>::T T;
        #pragma unroll
        for (int k = 0; k < KT; ++k) v[k] = az_i4{0, 0, 0, 0};
        if (rl >= st.n) return;
        const int bb = a.nb > 1 ? rl / a.S : 0, s = st.cell0 + rl - bb * a.S;
        const T* src = a.nchw ? (const T*)a.h + (size_t)(st.b0 + bb) * a.C * a.S + s : (const T*)a.h + (size_t)(st.rbase + rl) * a.C;
        const size_t cs = a.nchw ? a.S : 1;
        #pragma unroll
        for (int k = 0; k < KT; ++k) {
            const int c0 = k * KS + q * EP;
            if (k * KS >= a.C) break;
            T e[EP];
            if (c0 + EP <= a.C) {
                if (!a.nchw) {
                    if constexpr (DT == 0) *(az_f4*)e = *(const az_f4_u*)(src + c0);
                    else *(az_s8*)e = *(const az_s8_u*)(src + c0);
                } else {
                    #pragma unroll
                    for (int j = 0; j < EP; ++j) e[j] = src[(size_t)(c0 + j) * cs];
                }
            } else {
                #pragma unroll
                for (int j = 0; j < EP; ++j) e[j] = c0 + j < a.C ? src[(size_t)(c0 + j) * cs] : (T)0.f;
            }
            v[k] = *(az_i4*)e;
        }
    }
};

// Row statistics.  Four waves; a wave takes 16 rows of a step, all planes, and meets the others only where the board
// changes.  The features go from memory to fragments (no other wave wants these rows), the next tile's while this one is
// worked on.  Sparse targets: the tile's logits pass through LDS, half of the planes at a time where there are many, and
// the lanes pick out those that the entries name.
template <int DT, int OT, int CB> struct RowsCfg {
    static constexpr int PASSES = OT >= 6 ? 2 : 1, OTP = OT / PASSES, LDZ = OTP * 16 + 4;
    static constexpr size_t tile = (size_t)16 * LDZ * 4;             // of one wave
};
template <int DT, int OT, int CB> __global__ void __launch_bounds__(256, DT != 0 && CB == 1 ? 3 : DT == 0 && CB == 2 && OT >= 4 ? 1 : 2) az_policy_rows_kernel(PolicyDev a) {
    typedef Lay<DT, OT> L;
    typedef RowsCfg<DT, OT, CB> R;
    constexpr int NT = 256, KT = CB * 128 / L::KS;
    constexpr bool WLDS = w_in_lds<DT, OT, CB>();
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int Cp = (a.C + 31) / 32 * 32, ldc = Cp + L::EP;
    const Smem<DT, OT, CB, false> m(smem, a, Cp, a.counts ? 4 * R::tile : 0);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, q = lane >> 4, rl = wave * 16 + (lane & 15);
    float* zt = m.t + wave * (R::tile / 4);
    if (WLDS) stage_w<DT, OT>(a, m.w, Cp, tid, NT);
    for (int o = tid; o < OT * 16; o += NT) m.bias[o] = o < a.O ? az_load<DT>(a.bias, o) : 0.f;
    const int s_lo = (int)((long long)blockIdx.x * a.steps / gridDim.x), s_hi = (int)((long long)(blockIdx.x + 1) * a.steps / gridDim.x);
    RowFrags<DT, KT> f;
    f.load(a, step_at(a, s_lo), rl, q);
    int board = -1;
    for (int it = s_lo; it < s_hi; ++it) {
        const Step st = step_at(a, it);
        if (st.b0 != board) {
            if (a.legal || a.counts || board < 0) {
                __syncthreads();
                stage_boards(a, m.b, st.b0, tid, NT);
                __syncthreads();
            }
            board = st.b0;
        }
        az_f4 acc[OT];
        if (wave * 16 < st.n) {
            #pragma unroll
            for (int ot = 0; ot < OT; ++ot) acc[ot] = *(const az_f4*)(m.bias + ot * 16 + q * 4);
            #pragma unroll
            for (int k = 0; k < KT; ++k) {
                if (k * L::KS >= Cp) break;
                #pragma unroll
                for (int ot = 0; ot < OT; ++ot)
                    acc[ot] = az_mma<DT>(WLDS ? az_row_frag<DT>(m.w, ldc, ot * 16, k * L::KS, lane) : az_row_frag<DT>(a.wpad, Cp, ot * 16, k * L::KS, lane), f.v[k], acc[ot]);
            }
        }
        if (it + 1 < s_hi) f.load(a, step_at(a, it + 1), rl, q);
        if (wave * 16 >= st.n) continue;
        const int bb = a.nb > 1 ? rl / a.S : 0, s = st.cell0 + rl - bb * a.S, y = s / a.N;
        // entries that no action stands for: planes beyond the last, actions that are not allowed
        if (a.legal) {
            const unsigned bit = 1u << (s - y * a.N);
            const unsigned* words = m.b.words + (bb * a.N + (rl < st.n ? y : 0)) * (OT * 16) + q * 4;
            #pragma unroll
            for (int ot = 0; ot < OT; ++ot) {
                const az_i4 w = *(const az_i4*)(words + ot * 16);
                #pragma unroll
                for (int i = 0; i < 4; ++i) acc[ot][i] = (unsigned)w[i] & bit ? acc[ot][i] : -INFINITY;
            }
        }
        #pragma unroll
        for (int ot = 0; ot < OT; ++ot)
            if (ot * 16 + 16 > a.O) {
                #pragma unroll
                for (int i = 0; i < 4; ++i) if (ot * 16 + q * 4 + i >= a.O) acc[ot][i] = -INFINITY;
            }
        float tz = 0.f, tm = 0.f;
        // (an entry without a target does not count, whatever its logit; one with a target whose action is not allowed
        // gives -inf)
        if (!a.counts) {
            if (rl < st.n) {
                const float* dense = a.dense + ((size_t)(st.b0 + bb) * a.O + q * 4) * a.S + s;
                #pragma unroll
                for (int ot = 0; ot < OT; ++ot)
                    #pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (ot * 16 + q * 4 + i < a.O) {
                            const float tv = dense[(size_t)(ot * 16 + i) * a.S];
                            tz += tv != 0.f ? tv * acc[ot][i] : 0.f;
                            tm += tv;
                        }
            }
        } else {
            const int n = min(a.nb, a.B - st.b0) * a.cap, lo = st.cell0 + wave * 16, hi = min(lo + 16, st.cell0 + st.n);
            #pragma unroll
            for (int p = 0; p < R::PASSES; ++p) {
                #pragma unroll
                for (int j = 0; j < R::OTP; ++j) *(az_f4*)(zt + (lane & 15) * R::LDZ + j * 16 + q * 4) = acc[p * R::OTP + j];
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                // one board: every lane takes an entry, whichever row it names; several: a lane takes its own row's
                for (int e = a.nb > 1 ? q : lane; e < n; e += a.nb > 1 ? 4 : 64) {
                    int key;
                    float v = 0.f;
                    if (m.b.listed) key = m.b.key[e];
                    else key = entry_at(a, st, e, v);
                    const int row = key >> 8, o = (key & 255) - p * R::OTP * 16;
                    if (row >= lo && row < hi && (unsigned)o < (unsigned)(R::OTP * 16) && (a.nb == 1 || row == rl)) {
                        if (m.b.listed) v = m.b.val[e];
                        tz += v != 0.f ? v * zt[(row - lo) * R::LDZ + o] : 0.f;
                        tm += v;
                    }
                }
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
            }
        }
        float mx = -INFINITY;
        #pragma unroll
        for (int ot = 0; ot < OT; ++ot) mx = fmaxf(mx, fmaxf(fmaxf(acc[ot][0], acc[ot][1]), fmaxf(acc[ot][2], acc[ot][3])));
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));                      // four groups of lanes hold a row's planes
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float ml = mx == -INFINITY ? 0.f : mx * LOG2E;         // (a NaN logit is not the maximum, but its exponential joins the sum)
        float l = 0.f;
        #pragma unroll
        for (int ot = 0; ot < OT; ++ot)
            #pragma unroll
            for (int i = 0; i < 4; ++i) l += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[ot][i], LOG2E, -ml));
        for (int d = 16; d <= 32; d <<= 1) {
            l += __shfl_xor(l, d, 64);
            tz += __shfl_xor(tz, d, 64);
            tm += __shfl_xor(tm, d, 64);
        }
        if (q == 0 && rl < st.n) {                                   // (sparse, one board: tz and tm are the tile's entries' sums, spread over its rows)
            a.rowstat[st.rbase + rl] = az_f4{mx, l, tz, tm};
            asm volatile("s_nop 1");                                 // (a wide store reads its registers after it has issued)
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
        if (v[0] == -INFINITY) { l += v[1]; continue; }              // nothing allowed in the row: 0, or a NaN that stays
        if (v[0] <= m) l += v[1] * __builtin_amdgcn_exp2f((v[0] - m) * LOG2E);
        else { l = (m == -INFINITY ? l : l * __builtin_amdgcn_exp2f((m - v[0]) * LOG2E)) + v[1]; m = v[0]; }
    }
    float M = m;
    for (int d = 32; d > 0; d >>= 1) { const float om = __shfl_xor(M, d, 64); if (!(om <= M)) M = om; }
    l = m == -INFINITY ? l : l * __builtin_amdgcn_exp2f((m - M) * LOG2E);
    l = wave_sum(l);
    tz = wave_sum(tz);
    tm = wave_sum(tm);
    if (lane == 0) {
        const float lse = M == -INFINITY ? (l == l ? -INFINITY : l) : M + logf(l);
        const bool masked = tz == -INFINITY;                         // a target on an action that is not allowed
        const float loss = masked ? INFINITY : (tm != 0.f ? tm * lse : 0.f) - tz;
        a.stats[b] = az_f4{lse, tm, masked ? 1.f : 0.f, loss};
        if (a.loss) a.loss[b] = loss;
    }
}

// Gradients.  Eight waves.  A step: dz of 64 rows (16 rows and half of the planes a wave), then its product with w (32
// rows and a quarter of the channels a wave) and its product with the features (half of the planes and a quarter of the
// channels a wave, kept in registers over all of a workgroup's steps).  16-bit features: dz goes to LDS as hi + lo of the
// type, hi alone feeds dh (whose result is rounded to that type anyway), both feed dw (an fp32 sum over all rows: one
// rounding to 16 bits of each term would stay in it).
template <int DT, int OT, int CB> __global__ void __launch_bounds__(512) az_policy_grad_kernel(PolicyDev a) {
    typedef Lay<DT, OT> L;
    typedef typename AzElem<DT>::T T;
    constexpr int NT = 512, NP = CB * 128 / L::EP * ROWS / NT, OTH = (OT + 1) / 2, KO = L::OP / L::KS;
    constexpr int OG = OT > 1 ? 2 : 1, CG = 8 / OG, OTN = OT / OG, CTN = CB * 8 / CG;   // dw: groups of planes and channels, tiles of a wave
    constexpr bool WLDS = w_in_lds<DT, OT, CB>();
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int Cp = (a.C + 31) / 32 * 32, ldc = Cp + L::EP, pieces = Cp / L::EP;
    const Smem<DT, OT, CB, true> m(smem, a, Cp, L::z_bytes);
    float* t = m.t;                                                  // the step's targets, then its dz in the same place
    T* zhi = (T*)t;
    T* zlo = zhi + ROWS * L::LDO;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, q = lane >> 4, rt = wave & 3, half = wave >> 2;
    if (WLDS) stage_w<DT, OT>(a, m.w, Cp, tid, NT);
    for (int o = tid; o < OT * 16; o += NT) m.bias[o] = o < a.O ? az_load<DT>(a.bias, o) : 0.f;
    const int s_lo = (int)((long long)blockIdx.x * a.steps / gridDim.x), s_hi = (int)((long long)(blockIdx.x + 1) * a.steps / gridDim.x);
    const int og = OG == 2 ? wave & 1 : 0, cg = OG == 2 ? wave >> 1 : wave;
    az_f4 dw[CTN][OTN];
    #pragma unroll
    for (int i = 0; i < CTN; ++i)
        #pragma unroll
        for (int j = 0; j < OTN; ++j) dw[i][j] = az_f4{0.f, 0.f, 0.f, 0.f};
    az_f4 db[OTH];
    #pragma unroll
    for (int j = 0; j < OTH; ++j) db[j] = az_f4{0.f, 0.f, 0.f, 0.f};
    Feat<DT, NP> f;
    if (s_lo < s_hi) f.template load<NT>(a, step_at(a, s_lo), pieces, tid);
    // fp16: dz is r_b (a mean over the batch: 1 / B) times probabilities that may be 1e-5, below what fp16 resolves.  The
    // workgroup's dz carry a power of two that puts the largest r_b T_b of its boards at 2^9 .. 2^10; it comes off the
    // fp32 sums again.
    float up = 1.f, down = 1.f;
    if constexpr (DT == 1) {
        const Step first = step_at(a, s_lo), last = step_at(a, s_hi - 1);
        const int b1 = min(last.b0 + a.nb, a.B);
        float mx = 0.f;
        for (int b = first.b0 + tid; b < b1; b += NT) mx = fmaxf(mx, fabsf(a.scale * (a.row_scale ? a.row_scale[b] : 1.f) * a.stats[b][1]));
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
    int board = -1;
    for (int it = s_lo; it < s_hi; ++it) {
        const Step st = step_at(a, it);
        __syncthreads();                                             // the step before has read its LDS
        f.template store<NT>(a, m.h, Cp, pieces, tid);
        if (a.counts) for (int i = tid; i < ROWS * L::LDT / 4; i += NT) ((az_f4*)t)[i] = az_f4{0.f, 0.f, 0.f, 0.f};
        if (st.b0 != board) { stage_boards(a, m.b, st.b0, tid, NT); board = st.b0; }
        __syncthreads();
        if (it + 1 < s_hi) f.template load<NT>(a, step_at(a, it + 1), pieces, tid);
        const int rl = rt * 16 + (lane & 15);
        const bool live = rl < st.n;
        const int bb = live && a.nb > 1 ? rl / a.S : 0, b = st.b0 + bb, s = live ? st.cell0 + rl - bb * a.S : 0, y = s / a.N;
        const unsigned bit = 1u << (s - y * a.N);
        az_f4 tv[OTH];
        if (a.counts) {
            scatter_targets<L::LDT, 8>(a, m.b, t, st, wave, lane);
            __syncthreads();
            #pragma unroll
            for (int j = 0; j < OTH; ++j) {
                const int ot = half * OTH + j;
                tv[j] = ot < OT ? *(const az_f4*)(t + rl * L::LDT + ot * 16 + q * 4) : az_f4{0.f, 0.f, 0.f, 0.f};
            }
            __syncthreads();                                         // dz takes the targets' place
        } else {
            const float* dense = a.dense + ((size_t)b * a.O + half * OTH * 16 + q * 4) * a.S + s;
            #pragma unroll
            for (int j = 0; j < OTH; ++j)
                #pragma unroll
                for (int i = 0; i < 4; ++i) tv[j][i] = live && (half * OTH + j) * 16 + q * 4 + i < a.O ? dense[(size_t)(j * 16 + i) * a.S] : 0.f;
        }
        az_f4 acc[OTH];
        #pragma unroll
        for (int j = 0; j < OTH; ++j) acc[j] = half * OTH + j < OT ? *(const az_f4*)(m.bias + (half * OTH + j) * 16 + q * 4) : az_f4{0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < Cp; k += L::KS) {
            const az_i4 hb = az_row_frag<DT>(m.h, ldc, rt * 16, k, lane);
            #pragma unroll
            for (int j = 0; j < OTH; ++j) {
                const int ot = half * OTH + j;
                if (ot < OT) acc[j] = az_mma<DT>(WLDS ? az_row_frag<DT>(m.w, ldc, ot * 16, k, lane) : az_row_frag<DT>(a.wpad, Cp, ot * 16, k, lane), hb, acc[j]);
            }
        }
        const az_f4 bst = live ? a.stats[b] : az_f4{0.f, 0.f, 0.f, 0.f};
        const float rs = live ? up * (a.scale * (a.row_scale ? a.row_scale[b] : 1.f)) : 0.f;
        const float rT = rs * bst[1], lse2 = bst[0] * LOG2E;
        const unsigned* words = m.b.words + (bb * a.N + y) * (OT * 16) + half * OTH * 16 + q * 4;
        // one plane and no target outside the allowed actions: the bias moves every logit alike, its gradient is zero
        const bool bias_counts = a.O > 1 || bst[2] != 0.f;
        #pragma unroll
        for (int j = 0; j < OTH; ++j) {
            const int ot = half * OTH + j;
            if (ot * 16 >= L::OP) continue;
            az_f4 dz;
            #pragma unroll
            for (int i = 0; i < 4; ++i) dz[i] = rT * __builtin_amdgcn_exp2f(__builtin_fmaf(acc[j][i], LOG2E, -lse2)) - rs * tv[j][i];
            if (a.legal && ot < OT) {
                const az_i4 w = *(const az_i4*)(words + j * 16);
                #pragma unroll
                for (int i = 0; i < 4; ++i) dz[i] = (unsigned)w[i] & bit ? dz[i] : 0.f;
            }
            if (ot * 16 + 16 > a.O) {
                #pragma unroll
                for (int i = 0; i < 4; ++i) if (ot * 16 + q * 4 + i >= a.O) dz[i] = 0.f;
            }
            if (!live) dz = az_f4{0.f, 0.f, 0.f, 0.f};
            if (bias_counts) db[j] += dz;
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
        // dh: rows of a tile are channels, columns are cells
        {
            const int pair = wave & 1, cq = wave >> 1;
            az_i4 zf[2][KO];
            #pragma unroll
            for (int k = 0; k < KO; ++k)
                #pragma unroll
                for (int e = 0; e < 2; ++e) zf[e][k] = az_row_frag<DT>(zhi, L::LDO, (pair * 2 + e) * 16, k * L::KS, lane);
            #pragma unroll
            for (int j = 0; j < CB * 2; ++j) {
                const int ct = cq + 4 * j;
                if (ct * 16 >= Cp) continue;
                az_f4 d[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
                #pragma unroll
                for (int k = 0; k < KO; ++k) {
                    az_i4 wa;
                    if constexpr (WLDS) wa = az_col_frag<DT>(m.w, ldc, k * L::KS, ct * 16, lane);
                    else wa = az_row_frag<DT>(a.wpadt, L::OP, ct * 16, k * L::KS, lane);
                    d[0] = az_mma<DT>(wa, zf[0][k], d[0]);
                    d[1] = az_mma<DT>(wa, zf[1][k], d[1]);
                }
                const int c = ct * 16 + q * 4;
                #pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int row = (pair * 2 + e) * 16 + (lane & 15);
                    if (row >= st.n || c >= a.C) continue;
                    if constexpr (DT == 1) d[e] *= down;
                    if (!a.nchw) {
                        const size_t at = (size_t)(st.rbase + row) * a.C + c;
                        if (c + 4 <= a.C) {
                            if constexpr (DT == 0) *(az_f4_u*)((float*)a.dh + at) = d[e];
                            else *(az_s4_u*)((short*)a.dh + at) = az_s4{az_to16<DT>(d[e][0]), az_to16<DT>(d[e][1]), az_to16<DT>(d[e][2]), az_to16<DT>(d[e][3])};
                        } else for (int i = 0; i < 4; ++i) if (c + i < a.C) az_store<DT>(a.dh, at + i, d[e][i]);
                    } else {
                        const int b2 = a.nb > 1 ? row / a.S : 0, s2 = st.cell0 + row - b2 * a.S;
                        const size_t at = ((size_t)(st.b0 + b2) * a.C + c) * a.S + s2;
                        for (int i = 0; i < 4; ++i) if (c + i < a.C) az_store<DT>(a.dh, at + (size_t)i * a.S, d[e][i]);
                    }
                }
            }
        }
        // dw: rows of a tile are planes, columns are channels, the contraction runs over the step's rows (rows beyond the
        // step have dz = 0 and features of 0)
        #pragma unroll
        for (int k = 0; k < ROWS; k += L::KS) {
            if (k >= st.n) break;
            az_i4 zf[OTN][DT == 0 ? 1 : 2];
            #pragma unroll
            for (int j = 0; j < OTN; ++j) {
                zf[j][0] = az_col_frag<DT>(zhi, L::LDO, k, (og * OTN + j) * 16, lane);
                if constexpr (DT != 0) zf[j][1] = az_col_frag<DT>(zlo, L::LDO, k, (og * OTN + j) * 16, lane);
            }
            #pragma unroll
            for (int i = 0; i < CTN; ++i) {
                const int ct = cg + CG * i;
                if (ct * 16 >= Cp) continue;
                const az_i4 hb = az_col_frag<DT>(m.h, ldc, k, ct * 16, lane);
                #pragma unroll
                for (int j = 0; j < OTN; ++j) {
                    dw[i][j] = az_mma<DT>(zf[j][0], hb, dw[i][j]);
                    if constexpr (DT != 0) dw[i][j] = az_mma<DT>(zf[j][1], hb, dw[i][j]);
                }
            }
        }
    }
    float* out = a.partial + (size_t)blockIdx.x * ((size_t)a.O * a.C + a.O);
    #pragma unroll
    for (int i = 0; i < CTN; ++i) {
        const int c = (cg + CG * i) * 16 + (lane & 15);
        #pragma unroll
        for (int j = 0; j < OTN; ++j)
            #pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int o = (og * OTN + j) * 16 + q * 4 + e;
                if (o < a.O && c < a.C) out[(size_t)o * a.C + c] = dw[i][j][e] * down;
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
    const int Cp = (a.C + 31) / 32 * 32;
    const size_t lds = grad ? Smem<DT, OT, CB, true>::bytes(a, Cp, Lay<DT, OT>::z_bytes) : Smem<DT, OT, CB, false>::bytes(a, Cp, a.counts ? 4 * RowsCfg<DT, OT, CB>::tile : 0);
    const void* fn = grad ? (const void*)az_policy_grad_kernel<DT, OT, CB> : (const void*)az_policy_rows_kernel<DT, OT, CB>;
    if (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    if (grad) az_policy_grad_kernel<DT, OT, CB><<<groups, 512, lds, stream>>>(a);
    else {
        // as many workgroups as the chip holds: 160 KB of LDS a CU, at most four of four waves
        const int per_cu = lds * 4 <= LDS_BYTES ? 4 : (int)(LDS_BYTES / lds), room = 256 * per_cu;
        az_policy_rows_kernel<DT, OT, CB><<<a.steps < room ? a.steps : room, 256, lds, stream>>>(a);
    }
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

// how boards map to steps
void geometry(int B, int N, int& nb, int& blocks, long long& steps) {
    const int S = N * N;
    nb = S <= 32 ? (ROWS / S < MAX_BOARDS ? ROWS / S : MAX_BOARDS) : 1;
    blocks = nb > 1 ? 1 : (S + ROWS - 1) / ROWS;
    steps = nb > 1 ? ((long long)B + nb - 1) / nb : (long long)B * blocks;
}
// fp32 weights beyond LDS (w_in_lds): padded copies of at most 128 x 256
bool pads_weight(const az_policy_loss_args* p) { return p->dtype == AZ_F32 && p->C > 128 && p->c_out > 32; }
constexpr size_t PAD_BYTES = (size_t)128 * 256 * 4;

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
    int nb, blocks;
    long long steps;
    geometry(p->B, p->N, nb, blocks, steps);
    if (pads_weight(p)) n += 2 * PAD_BYTES;
    if (p->d_weight) n += up256((size_t)groups_of(steps) * ((size_t)p->c_out * p->C + p->c_out) * 4);
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
    long long steps;
    geometry(p->B, p->N, a.nb, a.blocks, steps);
    a.rows = a.B * a.S; a.steps = (int)steps;
    unsigned char* ws = (unsigned char*)workspace;
    a.rowstat = (az_f4*)ws; ws += up256((size_t)a.rows * sizeof(az_f4));
    a.stats = p->stats ? (az_f4*)p->stats : (az_f4*)ws; ws += up256((size_t)a.B * sizeof(az_f4));
    const bool pads = pads_weight(p);
    float* pad = (float*)ws;
    if (pads) { a.wpad = pad; a.wpadt = pad + PAD_BYTES / 4; ws += 2 * PAD_BYTES; }
    a.partial = (float*)ws;
    const int groups = groups_of(a.steps);
    hipError_t e = hipSuccess;
    if (a.B > 0 && pads) {
        az_policy_pad_weight_kernel<<<64, 256, 0, st>>>((const float*)p->weight, pad, pad + PAD_BYTES / 4, a.O, a.C, a.O <= 64 ? 64 : a.O <= 96 ? 96 : 128, (a.C + 31) / 32 * 32);
        e = hipGetLastError();
    }
    if (e == hipSuccess && a.B > 0 && !p->stats_given) {
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
