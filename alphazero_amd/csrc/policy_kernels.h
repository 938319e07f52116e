// policy_kernels.h -- the kernels of policy_loss.h, templates over the element type DT, planes OT (in 16s), channels CB (in
// 128s) and the way the features are read.
#pragma once
#include "policy_loss.h"

#include <type_traits>

namespace {

// dynamic LDS of the two product kernels
template <int DT, int OT, int CB> struct Lay {
    static constexpr int EP = AzElem<DT>::EP, KS = AzElem<DT>::KS, SZ = 16 / EP;
    static constexpr int OP = (OT * 16 + KS - 1) / KS * KS;          // planes, padded to a step of the contraction over them
    static constexpr int PAD = DT == 0 ? 4 : 16;                     // 16-bit rows: odd multiples of 32 bytes (az_col_frag), fp32: 16 bytes more
    static constexpr int LDT = OT * 16 + 4, LDO = OP + PAD;
    // channels are padded to what the kernel is built for: every LDS address is then a base and a constant
    // LDW: rows of w, read along only, 16 in one go: an odd multiple of 16 bytes
    static constexpr int CP = CB * 128, LDC = CP + PAD, LDW = CP + EP, PIECES = CP / EP;
    static constexpr size_t w_bytes = (size_t)OP * LDW * SZ, h_bytes = (size_t)ROWS * LDC * SZ;
    static constexpr size_t z_bytes = (size_t)ROWS * (LDO > LDT ? LDO : LDT) * 4;
};

__device__ __forceinline__ float wave_max(float x) {
    for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o, 64));
    return x;
}

// How the features are read.  A load that is to stay in flight is unconditional, its address clamped into the tensor, and
// what it should not have brought is dropped where it is used.
//   WHOLE_LAST   channels last, C a multiple of a product step (32; fp32: 16): 16-byte loads
//   WHOLE_FIRST  channels first, C such a multiple: one element a load, neighbouring lanes neighbouring cells
//   ANY          anything else: one element a load, every index clamped
enum { WHOLE_LAST, WHOLE_FIRST, ANY };

// The kernel's arguments, read again from the argument segment: called at the top of a loop's body, what is derived from
// them does not have to live through the whole loop (it would fill the scalar registers, and spill into vector ones).
__device__ __forceinline__ PolicyDev arguments() {
    typedef const __attribute__((address_space(4))) PolicyDev* Args;
    Args p = (Args)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const PolicyDev*)p;
}

// A value the compiler may not carry over from an earlier iteration: index arithmetic of the one-element loads is done
// anew for each tile instead of filling the registers.
__device__ __forceinline__ int anew(int x) { asm volatile("" : "+v"(x)); return x; }
__device__ __forceinline__ int anew_s(int x) { asm volatile("" : "+s"(x)); return x; }      // (of a wave-uniform value)

// (policy_loss.hip: az_policy_pad_weight_kernel)
template <int DT, int OT, int CB> __host__ __device__ constexpr bool w_in_lds() { return !(DT == 0 && CB == 2 && OT >= 4); }

// w [O][C] -> LDS [OP][Cp + EP], zero beyond O and C, in pieces of 16 bytes; eight loads of a thread in flight
template <int DT, int OT, int CB> __device__ __forceinline__ void stage_w(const PolicyDev& a, void* wl, int tid) {
    typedef Lay<DT, OT, CB> L;
    typedef typename AzElem<DT>::T T;
    constexpr int EP = L::EP, U = 8;
    constexpr int per = L::PIECES, total = L::OP * per;
    for (int base = tid; base < total; base += NT * U) {
        az_i4 v[U];
        if (a.C % EP == 0) {
            #pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = min(base + u * NT, total - 1), o = i / per, c = (i - o * per) * EP;
                const T* src = (const T*)a.w + (size_t)min(o, a.O - 1) * a.C + min(c, a.C - EP);
                if constexpr (DT == 0) v[u] = __builtin_bit_cast(az_i4, *(const az_f4_u*)src);
                else v[u] = __builtin_bit_cast(az_i4, *(const az_s8_u*)src);
            }
        } else {
            #pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = min(base + u * NT, total - 1), o = i / per, c = (i - o * per) * EP;
                const T* src = (const T*)a.w + (size_t)min(o, a.O - 1) * a.C;
                T e[EP];
                #pragma unroll
                for (int k = 0; k < EP; ++k) { const T x = src[min(c + k, a.C - 1)]; e[k] = c + k < a.C ? x : (T)0.f; }
                v[u] = *(az_i4*)e;
            }
        }
        #pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = base + u * NT, o = i / per, c = (i - o * per) * EP;
            if (i < total) *(az_i4*)((char*)wl + ((size_t)o * L::LDW + c) * L::SZ) = o < a.O && c < a.C ? v[u] : az_i4{0, 0, 0, 0};
        }
    }
}

// What a workgroup's boards need beside the features, brought to LDS when the board changes: the legal-move words as
// [board, row][plane], and the sparse targets sorted by blocks of 64 rows as {row of the boards * 256 + plane, value}.
constexpr int BLOCKS = 16;                                           // blocks of 64 rows: boards of 32 x 32
struct BoardLds {
    unsigned* words;                                                 // bit 0 = no action stands for the entry: a plane beyond the last, or not allowed
    int planes;                                                      // words of a line: the planes, padded to 16
    int* key;
    float* val;
    int* cnt;                                                        // [64-entry chunk][BLOCKS]
    int* start;                                                      // [BLOCKS + 1]: a block's first entry
    az_f4* stat;                                                     // [MAX_BOARDS] of the gradients: {max z, r T / sum of exp, r, is the loss infinite or the gradient NaN}
    bool listed;                                                     // the entries fit
};
// entries outside the board's actions: -1
__device__ __forceinline__ int entry_key(const PolicyDev& a, int act, int bb) {
    if ((unsigned)act >= (unsigned)(a.O * a.S)) return -1;
    const int o = act / a.S;
    return (bb * a.S + act - o * a.S) * 256 + o;
}
__device__ __forceinline__ int entry_at(const PolicyDev& a, int b0, int e, float& v) {
    const int bb = a.nb > 1 ? e / a.cap : 0, k = e - bb * a.cap;
    const size_t at = (size_t)(b0 + bb) * a.cap + k;
    if (k >= a.counts[b0 + bb]) return -1;
    v = a.probs[at];
    return entry_key(a, a.actions[at], bb);
}

// The words before any board's are there: without legal-move words every action of the planes there are is allowed.
__device__ __forceinline__ void init_words(const PolicyDev& a, const BoardLds& l, int tid) {
    for (int i = tid; i < a.nb * a.N * l.planes; i += NT) l.words[i] = !a.legal && i % l.planes < a.O ? ~0u : 0u;
}

// One group's words and entries: a thread's first loads go out together.
template <bool GRAD> struct BoardLoads {
    static constexpr int W = 4, E = ENTRIES / NT;
    unsigned w[W];
    int act[E], cnt[E];
    float val[E];
    az_f4 st;
    float r;
    __device__ __forceinline__ void load(const PolicyDev& a, const BoardLds& l, int b0, int tid) {
        const int boards = min(a.nb, a.B - b0), b = b0 + min(tid, boards - 1);
        if (GRAD) { st = a.stats[b]; r = a.row_scale ? a.row_scale[b] : 1.f; }
        if (a.legal) {
            const int n = boards * a.O * a.N;
            const unsigned* src = a.legal + (size_t)b0 * a.O * a.N;
            #pragma unroll
            for (int u = 0; u < W; ++u) w[u] = src[min(tid + u * NT, n - 1)];
        }
        if (l.listed) {
            const int n = boards * a.cap;
            #pragma unroll
            for (int u = 0; u < E; ++u) {
                const int e = min(tid + u * NT, n - 1);
                cnt[u] = a.counts[b0 + (a.nb > 1 ? e / a.cap : 0)];
                act[u] = a.actions[(size_t)b0 * a.cap + e];
                val[u] = a.probs[(size_t)b0 * a.cap + e];
            }
        }
    }
    __device__ __forceinline__ void put_word(const PolicyDev& a, const BoardLds& l, int i, unsigned v) const {
        const int bo = (int)((unsigned)i * a.mag_w >> 20), y = i - bo * a.N, bb = a.nb > 1 ? bo / a.O : 0;
        l.words[(bb * a.N + y) * l.planes + bo - bb * a.O] = v;
    }
    // every thread; ends in a barrier
    __device__ __forceinline__ void store(const PolicyDev& a, const BoardLds& l, int b0, int tid) const {
        const int boards = min(a.nb, a.B - b0), lane = tid & 63, wave = tid >> 6;
        if (GRAD && tid < boards) {
            const float rs = a.scale * r;
            const float rp = rs * st[1] * st[2];
            l.stat[tid] = az_f4{st[0], rp, rs, st[3] < 0.f || !(fabsf(rp) < INFINITY) ? 1.f : 0.f};
        }
        if (a.legal) {
            const int n = boards * a.O * a.N;
            #pragma unroll
            for (int u = 0; u < W; ++u) if (tid + u * NT < n) put_word(a, l, tid + u * NT, w[u]);
            const unsigned* src = a.legal + (size_t)b0 * a.O * a.N;
            for (int i = tid + W * NT; i < n; i += NT) put_word(a, l, i, src[i]);
        }
        if (l.listed) {
            // a stable counting sort by block: the entries of a block keep their order, whatever the waves' timing
            const int n = boards * a.cap, chunks = (n + 63) / 64, blocks = (boards * a.S + 63) / 64;
            int key[E], rank[E];
            #pragma unroll
            for (int u = 0; u < E; ++u) {
                const int e = tid + u * NT, chunk = wave + u * WAVES;
                const int bb = a.nb > 1 ? min(e, n - 1) / a.cap : 0;
                key[u] = e < n && e - bb * a.cap < cnt[u] ? entry_key(a, act[u], bb) : -1;
                if (chunk >= chunks) continue;
                const int block = key[u] < 0 ? -1 : key[u] >> 14;
                int mine = 0;
                for (int t = 0; t < blocks; ++t) {
                    const unsigned long long m = __ballot(block == t);
                    if (block == t) rank[u] = __popcll(m & ((1ull << lane) - 1));
                    if (lane == t) mine = __popcll(m);
                }
                if (lane < BLOCKS) l.cnt[chunk * BLOCKS + lane] = mine;
            }
            __syncthreads();
            // lane t of every wave: where block t starts, and within it this wave's chunks
            int sum = 0, before[E] = {};
            for (int c = 0; c < chunks; ++c) {
                const int k = lane < BLOCKS ? l.cnt[c * BLOCKS + lane] : 0;
                #pragma unroll
                for (int u = 0; u < E; ++u) before[u] += c < wave + u * WAVES ? k : 0;
                sum += k;
            }
            int incl = sum;
            for (int d = 1; d < BLOCKS; d <<= 1) { const int o = __shfl_up(incl, d, 64); if (lane >= d) incl += o; }
            if (wave == 0 && lane < BLOCKS) { l.start[lane] = incl - sum; if (lane == BLOCKS - 1) l.start[BLOCKS] = incl; }
            #pragma unroll
            for (int u = 0; u < E; ++u) {
                const int at = __shfl(incl - sum + before[u], key[u] < 0 ? 0 : key[u] >> 14, 64) + rank[u];
                if (key[u] >= 0) {
                    l.key[at] = key[u];
                    l.val[at] = val[u];
                }
            }
        }
        __syncthreads();
    }
};

template <bool GRAD> __device__ __forceinline__ void stage_boards(const PolicyDev& a, const BoardLds& l, int b0, int tid) {
    BoardLoads<GRAD> x;
    x.load(a, l, b0, tid);
    x.store(a, l, b0, tid);
}

// The gradient kernel's boards in turn; the loads of the one to come wait in registers.
struct BoardQueue {
    BoardLoads<true> x;
    // first: any board; next: the one behind, which is on its way
    __device__ __forceinline__ void first(const PolicyDev& a, const BoardLds& l, int b0, int tid) {
        x.load(a, l, b0, tid);
        x.store(a, l, b0, tid);
        if (b0 + a.nb < a.B) x.load(a, l, b0 + a.nb, tid);
    }
    __device__ __forceinline__ void next(const PolicyDev& a, const BoardLds& l, int b0, int tid) {
        x.store(a, l, b0, tid);
        if (b0 + a.nb < a.B) x.load(a, l, b0 + a.nb, tid);
    }
};

// LDS of the product kernels, in this order; zb: bytes of the kernel's own tile (logits or dz)
template <int DT, int OT, int CB, int HBUF, bool WBUF> struct Smem {
    typedef Lay<DT, OT, CB> L;
    unsigned char *w, *h;
    float *t, *bias;
    BoardLds b;
    __device__ __forceinline__ Smem(unsigned char* p, const PolicyDev& a, size_t zb) {
        w = p; p += WBUF ? L::w_bytes : 0;
        h = p; p += HBUF * L::h_bytes;
        t = (float*)p; p += zb;
        bias = (float*)p; p += OT * 16 * 4;
        b.stat = (az_f4*)p; p += MAX_BOARDS * 16;
        b.words = (unsigned*)p; p += (size_t)a.nb * a.N * OT * 16 * 4;
        b.planes = OT * 16;
        const int room = a.room;
        b.listed = room > 0;
        b.key = (int*)p; p += (size_t)room * 4;
        b.val = (float*)p; p += (size_t)room * 4;
        b.start = (int*)p; p += (BLOCKS + 1) * 4;
        b.cnt = (int*)p;
    }
    static size_t bytes(const PolicyDev& a, size_t zb) {
        const size_t room = a.room;
        return (WBUF ? L::w_bytes : 0) + HBUF * L::h_bytes + zb + OT * 16 * 4 + MAX_BOARDS * 16 + (size_t)a.nb * a.N * OT * 16 * 4 +
               (room ? room * 8 + (BLOCKS + 1) * 4 + (room + 63) / 64 * BLOCKS * 4 : 0);
    }
};

// Running {max, sum of exp} of a set of logits, joined.  Nothing in it yet: {-inf, 0}; a NaN logit is not the maximum, but
// its exponential joins the sum.
__device__ __forceinline__ float rescale(float m, float to) { return m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - to) * LOG2E); }
__device__ __forceinline__ void join(float& m, float& l, float om, float ol) {
    const float to = fmaxf(m, om);
    l = l * rescale(m, to) + ol * rescale(om, to);
    m = to;
}
// A whole wave.  Where a NaN made the targets' sum one, the loss takes the sum of the others; where one is negative (fp16), the
// gradients need the sum of the magnitudes: the targets are read once more.  So they are where a target outside the allowed
// actions may be a negative one: tz is then +inf, or NaN beside a positive one, instead of -inf.
template <int DT> __device__ __forceinline__ void finish_board(const PolicyDev& a, int b, float m, float l, float tz, float tm, bool negative, int lane) {
    float tl = tm, ta = tm;
    bool masked = tz == -INFINITY;                                   // a target on an action that is not allowed
    const bool odd = a.legal && !masked && !(fabsf(tz) < INFINITY);
    if (tm != tm || negative || odd) {
        float sum = 0.f, all = 0.f;
        const int n = a.counts ? min(a.counts[b], a.cap) : a.O * a.S;
        for (int i = lane; i < n; i += 64) {
            const float v = a.counts ? a.probs[(size_t)b * a.cap + i] : a.dense[(size_t)b * a.O * a.S + i];
            const int act = a.counts ? a.actions[(size_t)b * a.cap + i] : i;
            if (!__builtin_islessgreater(v, 0.f) || (unsigned)act >= (unsigned)(a.O * a.S)) continue;
            sum += v;
            all += fabsf(v);
            if (odd) {
                const int line = act / a.N, x = act - line * a.N;    // (plane, row)
                masked |= !(a.legal[(size_t)b * a.O * a.N + line] >> x & 1);
            }
        }
        masked = __ballot(masked) != 0;
        for (int o = 32; o > 0; o >>= 1) { sum += __shfl_xor(sum, o, 64); all += __shfl_xor(all, o, 64); }
        if (tm != tm) tl = sum;
        ta = all;
    }
    if (lane != 0) return;
    const float lse = m == -INFINITY ? (l == l ? -INFINITY : l) : m + logf(l);
    const float mag = DT == 1 ? ta : 1.f;
    const float loss = masked ? INFINITY : (tl != 0.f ? tl * lse : 0.f) - tz;
    // The gradients take probabilities as exp2((z - max) log2 e) / l, which is exactly 1 where one action is allowed: an lse rounded to 32 bits, off by up to 2^-22
    // where it is about 5, would move all of a board's probabilities one way, and where one plane's sum to the targets' sum
    // that is what is left of the products with features of one sign.
    a.stats[b] = az_f4{m == -INFINITY ? 0.f : m, tm, l == 0.f ? 0.f : 1.f / l, masked ? -mag : mag};
    if (a.loss) a.loss[b] = loss;
}

// Fragments of 16 rows of the features straight from memory, all channels.  Rows beyond the last are the last one again
// (nobody reads their columns of the product).
template <int DT, int KT, int MODE> struct RowFrags {
    az_i4 v[KT];
    __device__ __forceinline__ void load(const PolicyDev& a, int b0, int row, int rows, int q) {
        constexpr int EP = AzElem<DT>::EP, KS = AzElem<DT>::KS;
        typedef typename AzElem<DT>::T T;
        row = min(row, rows - 1);
        const T* group = (const T*)a.h + (size_t)b0 * a.S * a.C;
        const int bb = MODE != WHOLE_LAST && a.nb > 1 ? (int)((unsigned)row * a.mag_s >> 16) : 0;
        if constexpr (MODE == WHOLE_LAST) {
            const int at = row * a.C + q * EP;
            #pragma unroll
            for (int k = 0; k < KT; ++k) {
                const T* p = group + min(k * KS, a.C - KS) + at;
                if constexpr (DT == 0) v[k] = __builtin_bit_cast(az_i4, *(const az_f4_u*)p);
                else v[k] = __builtin_bit_cast(az_i4, *(const az_s8_u*)p);
            }
        } else if constexpr (MODE == WHOLE_FIRST) {
            const int at = anew(bb * (a.C - 1) * a.S + row + q * EP * a.S), S = anew_s(a.S);
            #pragma unroll
            for (int k = 0; k < KT; ++k) {
                T e[EP];
                #pragma unroll
                for (int j = 0; j < EP; ++j) e[j] = (group + (min(k * KS, a.C - KS) + j) * S)[at];
                v[k] = *(az_i4*)e;
            }
        } else {
            const int cs = anew_s(a.nchw ? a.S : 1), at = a.nchw ? bb * (a.C - 1) * a.S + row : row * a.C, c0 = anew(q * EP);
            #pragma unroll
            for (int k = 0; k < KT; ++k) {
                T e[EP];
                #pragma unroll
                for (int j = 0; j < EP; ++j) e[j] = group[at + min(c0 + k * KS + j, a.C - 1) * cs];
                v[k] = *(az_i4*)e;
            }
        }
    }
    // channels beyond the last are zero
    __device__ __forceinline__ az_i4 frag(const PolicyDev& a, int k, int q) const {
        constexpr int EP = AzElem<DT>::EP, KS = AzElem<DT>::KS;
        typedef typename AzElem<DT>::T T;
        if (MODE != ANY) return v[k];
        T e[EP];
        *(az_i4*)e = v[k];
        const int c0 = k * KS + q * EP;
        #pragma unroll
        for (int j = 0; j < EP; ++j) e[j] = c0 + j < a.C ? e[j] : (T)0.f;
        return *(az_i4*)e;
    }
};

// acc += w h over the channels: step(k, w) multiplies the fragments that fetch(k, w) brings.  All KT steps of the width
// the kernel is built for as straight code (the LDS reads run ahead of the products by themselves); fewer under checks.
// AHEAD: the fragments come from memory, so they are asked for one step early, and no earlier (all at once they would
// take more registers than there are).
template <int KT, int KS, int W, bool AHEAD, class F, class S> __device__ __forceinline__ void product(int C, const F& fetch, const S& step) {
    if constexpr (AHEAD) {
        az_i4 w[2][W];
        fetch(0, w[0]);
        #pragma unroll
        for (int k = 0; k < KT; ++k) {
            if (k * KS < C) {
                if (k + 1 < KT) fetch(k + 1, w[(k + 1) & 1]);        // (the padded copy is as wide as the kernel)
                step(k, w[k & 1]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    } else if (C > (KT - 1) * KS) {
        #pragma unroll
        for (int k = 0; k < KT; ++k) { az_i4 w[W]; fetch(k, w); step(k, w); }
    } else {
        #pragma unroll
        for (int k = 0; k < KT - 1; ++k)
            if (k * KS < C) { az_i4 w[W]; fetch(k, w); step(k, w); }
    }
}

// Losses.  A workgroup takes a board (or nb small ones) at a time, its waves the tiles of 16 rows in turn, all planes.  The
// features go from memory to fragments (no other wave wants these rows), the next tile's while this one is worked on; the
// waves meet only where the board changes.  Planes are taken half at a time from 64 on (all at
// once leaves a wave too few registers for four waves a SIMD: 512 boards of 20 x 20, 128 planes bf16 76 us, in halves 40;
// 91 planes 33 and 30, 64 planes 23.5 and 24).  Sparse targets: the logits pass through LDS, and lanes
// pick out those that the tile's entries name.
// 2048 boards of 20 x 20, 128 channels, 91 planes fp16, legal actions only: 88 us, 2.6 TB/s of the features (43 us of copying).
// By counters the vector units issue for 60 % of that (24 instructions a logit: exponential, mask, maximum, and their share of
// addresses and conversions), the matrix units work for 10 %; a wave's loads, products and exponentials follow one another, and
// what four waves a SIMD do not hide of that is the rest.  4096 boards of 15 x 15, one plane bf16: 61 us,
// 3.9 TB/s, bound by memory.  256 boards of 20 x 20, 256 channels fp32: 91 us, 52 TFLOP/s.
template <int OT> struct LossTile {
    static constexpr int PASSES = OT >= 4 ? 2 : 1, OTP = OT / PASSES, LDZ = OTP * 16 + 4;
    static constexpr size_t bytes = (size_t)16 * LDZ * 4;            // of one wave
};
template <int DT, int OT, int CB> __host__ __device__ constexpr int loss_waves() { return DT != 0 && CB == 1 ? 4 : 2; }   // a SIMD
template <int DT, int OT, int CB, int MODE> __global__ void __launch_bounds__(NT, (loss_waves<DT, OT, CB>())) az_policy_loss_kernel(PolicyDev a, int groups) {
    typedef Lay<DT, OT, CB> L;
    typedef LossTile<OT> R;
    constexpr int KT = CB * 128 / L::KS;
    constexpr bool WLDS = w_in_lds<DT, OT, CB>();
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    __shared__ az_f4 red[4 * ROWS];
    __shared__ int negative[MAX_BOARDS];                             // fp16: has the board a negative target
    constexpr int Cp = L::CP;
    const Smem<DT, OT, CB, 0, WLDS> m(smem, a, a.counts ? WAVES * R::bytes : 0);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, q = lane >> 4;
    float* zt = m.t + wave * (R::bytes / 4);
    const int g_lo = (int)((long long)blockIdx.x * groups / gridDim.x), g_hi = (int)((long long)(blockIdx.x + 1) * groups / gridDim.x);
    RowFrags<DT, KT, MODE> f;
    f.load(a, g_lo * a.nb, wave * 16 + (lane & 15), min(a.nb, a.B - g_lo * a.nb) * a.S, q);
    if (WLDS) stage_w<DT, OT, CB>(a, m.w, tid);
    for (int o = tid; o < OT * 16; o += NT) m.bias[o] = o < a.O ? az_load<DT>(a.bias, o) : 0.f;
    init_words(a, m.b, tid);
    if (tid < MAX_BOARDS) negative[tid] = 0;
    __syncthreads();
    for (int g = g_lo; g < g_hi; ++g) {
        const int b0 = g * a.nb, rows = min(a.nb, a.B - b0) * a.S;
        stage_boards<false>(a, m.b, b0, tid);
        float mx = -INFINITY, l = 0.f, tz = 0.f, tm = 0.f;
        #pragma unroll 1
        for (int r0 = wave * 16; r0 < rows; r0 += WAVES * 16) {
            const PolicyDev a = arguments();
            const int rl = r0 + (lane & 15);
            const bool live = rl < rows;
            const int bb = live && a.nb > 1 ? (int)((unsigned)rl * a.mag_s >> 16) : 0, s = live ? rl - bb * a.S : 0, y = (int)((unsigned)s * a.mag_n >> 16);
            const unsigned bit = live ? 1u << (s - y * a.N) : 0u;
            const unsigned* words = m.b.words + (bb * a.N + y) * (OT * 16) + q * 4;
            const float* dense = a.dense + (size_t)b0 * a.O * a.S;
            const int hi = min(r0 + 16, rows), e0 = m.b.listed ? m.b.start[r0 >> 6] : 0, e1 = m.b.listed ? m.b.start[(r0 >> 6) + 1] : min(a.nb, a.B - b0) * a.cap;
            int key0 = -1;
            float val0 = 0.f;
            if (m.b.listed && e0 + lane < e1) { key0 = m.b.key[e0 + lane]; val0 = m.b.val[e0 + lane]; }
            #pragma unroll 1
            for (int o0 = 0; o0 < OT * 16; o0 += R::OTP * 16) {      // planes o0 .. o0 + 16 OTP - 1
                // loads return in order: the targets are asked for ahead of the next tile's features
                float tv[R::OTP][4];
                if (!a.counts) {
                    const int at = (bb * a.O + o0 + q * 4) * a.S + s, last = ((bb + 1) * a.O - 1) * a.S + s;
                    #pragma unroll
                    for (int j = 0; j < R::OTP; ++j)
                        #pragma unroll
                        for (int i = 0; i < 4; ++i) tv[j][i] = dense[min(at + (j * 16 + i) * a.S, last)];
                }
                az_f4 acc[R::OTP];
                #pragma unroll
                for (int j = 0; j < R::OTP; ++j) acc[j] = *(const az_f4*)(m.bias + o0 + j * 16 + q * 4);
                const auto step = [&](int k, const az_i4* w) __attribute__((always_inline)) {
                    const az_i4 hb = f.frag(a, k, q);
                    #pragma unroll
                    for (int j = 0; j < R::OTP; ++j) acc[j] = az_mma<DT>(w[j], hb, acc[j]);
                };
                const auto fetch = [&](int k, az_i4* w) __attribute__((always_inline)) {
                    #pragma unroll
                    for (int j = 0; j < R::OTP; ++j) w[j] = WLDS ? az_row_frag<DT>(m.w, L::LDW, o0 + j * 16, k * L::KS, lane) : az_row_frag<DT>(a.wpad, Cp, o0 + j * 16, k * L::KS, lane);
                };
                product<KT, L::KS, R::OTP, !WLDS>(a.C, fetch, step);
                // the wave's next tile: of this group, or the first of the next one (which the barriers between do not touch)
                if (o0 + R::OTP * 16 >= OT * 16) {
                    if (r0 + WAVES * 16 < rows) f.load(a, b0, rl + WAVES * 16, rows, q);
                    else if (g + 1 < g_hi) f.load(a, b0 + a.nb, wave * 16 + (lane & 15), min(a.nb, a.B - b0 - a.nb) * a.S, q);
                }
                #pragma unroll
                for (int j = 0; j < R::OTP; ++j) {
                    const az_i4 w = *(const az_i4*)(words + o0 + j * 16);
                    #pragma unroll
                    for (int i = 0; i < 4; ++i) acc[j][i] = (unsigned)w[i] & bit ? acc[j][i] : -INFINITY;
                }
                // (an entry without a target does not count, whatever its logit; one with a target whose action is not
                // allowed gives -inf; a NaN is no target for the loss: finish_board)
                if (!a.counts) {
                    float least = 0.f;
                    #pragma unroll
                    for (int j = 0; j < R::OTP; ++j)
                        #pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float v = live && o0 + j * 16 + q * 4 + i < a.O ? tv[j][i] : 0.f;
                            tz += __builtin_islessgreater(v, 0.f) ? v * acc[j][i] : 0.f;
                            tm += v;
                            least = fminf(least, v);
                        }
                    if (DT == 1 && least < 0.f) negative[bb] = 1;
                } else {
                    #pragma unroll
                    for (int j = 0; j < R::OTP; ++j) *(az_f4*)(zt + (lane & 15) * R::LDZ + j * 16 + q * 4) = acc[j];
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    __builtin_amdgcn_wave_barrier();
                    const auto take = [&](int k, float v) __attribute__((always_inline)) {
                        const int row = (k >> 8) - r0, o = (k & 255) - o0;
                        if ((unsigned)row < (unsigned)(hi - r0) && (unsigned)o < (unsigned)(R::OTP * 16)) {
                            tz += __builtin_islessgreater(v, 0.f) ? v * zt[row * R::LDZ + o] : 0.f;
                            tm += v;
                            if (DT == 1 && v < 0.f) negative[bb] = 1;
                        }
                    };
                    if (m.b.listed && a.nb == 1) {                   // every lane takes an entry, whichever row it names
                        take(key0, val0);
                        for (int e = e0 + 64 + lane; e < e1; e += 64) take(m.b.key[e], m.b.val[e]);
                    } else                                           // several boards: a lane takes its own row's
                        for (int e = e0 + (a.nb > 1 ? q : lane); e < e1; e += a.nb > 1 ? 4 : 64) {
                            float v = 0.f;
                            int k;
                            if (m.b.listed) { k = m.b.key[e]; v = m.b.val[e]; } else k = entry_at(a, b0, e, v);
                            if (k >= 0 && (a.nb == 1 || k >> 8 == rl)) take(k, v);
                        }
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    __builtin_amdgcn_wave_barrier();
                }
                float to = mx;
                #pragma unroll
                for (int j = 0; j < R::OTP; ++j) to = fmaxf(to, fmaxf(fmaxf(acc[j][0], acc[j][1]), fmaxf(acc[j][2], acc[j][3])));
                const float ml = to == -INFINITY ? 0.f : to;
                l *= rescale(mx, to);
                #pragma unroll
                for (int j = 0; j < R::OTP; ++j)
                    #pragma unroll
                    for (int i = 0; i < 4; ++i) l += __builtin_amdgcn_exp2f((acc[j][i] - ml) * LOG2E);
                mx = to;
            }
        }
        if (a.nb == 1) {
            for (int d = 32; d > 0; d >>= 1) {
                join(mx, l, __shfl_xor(mx, d, 64), __shfl_xor(l, d, 64));
                tz += __shfl_xor(tz, d, 64);
                tm += __shfl_xor(tm, d, 64);
            }
            if (lane == 0) red[wave] = az_f4{mx, l, tz, tm};
        } else if (wave < 4) red[wave * 64 + (lane & 15) * 4 + q] = az_f4{mx, l, tz, tm};
        __syncthreads();
        if (a.nb == 1) {
            if (wave == 0) {
                az_f4 r = red[0];
                float fm = r[0], fl = r[1], fz = r[2], ft = r[3];
                for (int w = 1; w < WAVES; ++w) { r = red[w]; join(fm, fl, r[0], r[1]); fz += r[2]; ft += r[3]; }
                const bool neg = DT == 1 && negative[0];             // (nobody sets it again before the next board's barriers)
                if (DT == 1 && lane == 0) negative[0] = 0;
                finish_board<DT>(a, b0, fm, fl, fz, ft, neg, lane);
            }
        } else
            for (int bb = wave; bb * a.S < rows; bb += WAVES) {
                float fm = -INFINITY, fl = 0.f, fz = 0.f, ft = 0.f;
                for (int i = lane; i < a.S * 4; i += 64) { const az_f4 r = red[bb * a.S * 4 + i]; join(fm, fl, r[0], r[1]); fz += r[2]; ft += r[3]; }
                for (int d = 32; d > 0; d >>= 1) {
                    join(fm, fl, __shfl_xor(fm, d, 64), __shfl_xor(fl, d, 64));
                    fz += __shfl_xor(fz, d, 64);
                    ft += __shfl_xor(ft, d, 64);
                }
                const bool neg = DT == 1 && negative[bb];
                if (DT == 1 && lane == 0) negative[bb] = 0;
                finish_board<DT>(a, b0 + bb, fm, fl, fz, ft, neg, lane);
            }
    }
}

// A step of the gradients: up to 64 rows, a block of a board or whole boards; cells cell0 .. of board b0.
struct Step {
    int b0, blk, cell0, rows;
    __device__ __forceinline__ void set(const PolicyDev& a) {
        cell0 = blk * ROWS;
        rows = a.nb > 1 ? min(a.nb, a.B - b0) * a.S : min(ROWS, a.S - cell0);
    }
    __device__ __forceinline__ Step(const PolicyDev& a, int it) {
        const int g = it / a.blocks;
        b0 = g * a.nb; blk = it - g * a.blocks;
        set(a);
    }
    __device__ __forceinline__ void next(const PolicyDev& a) {
        if (++blk == a.blocks) { blk = 0; b0 += a.nb; }
        set(a);
    }
};

// The 16-byte pieces of a step's features that a thread carries from memory to LDS.  WHOLE_LAST: consecutive threads take
// consecutive pieces of a row; otherwise a wave takes one piece of all 64 rows.
template <int DT, int NP, int MODE, int NW = WAVES> struct Feat {                // NW: waves that take part
    static constexpr int pieces = NP * NW, LDC = pieces * AzElem<DT>::EP + (DT == 0 ? 4 : 16);
    az_i4 v[NP];
    __device__ __forceinline__ void place(int i, int tid, int& row, int& p) const {
        const int k = tid + i * NW * 64;
        if constexpr (MODE == WHOLE_LAST) { row = k / pieces; p = k - row * pieces; }
        else { row = tid & (ROWS - 1); p = __builtin_amdgcn_readfirstlane(tid / ROWS) + i * NW; }
    }
    __device__ __forceinline__ void load(const PolicyDev& a, const Step& st, int tid) {
        constexpr int EP = AzElem<DT>::EP;
        typedef typename AzElem<DT>::T T;
        const bool first = MODE == WHOLE_FIRST || (MODE == ANY && a.nchw);
        const T* group = (const T*)a.h + (size_t)st.b0 * a.S * a.C + (first ? st.cell0 : st.cell0 * a.C);
        #pragma unroll
        for (int i = 0; i < NP; ++i) {
            int row, p;
            place(i, tid, row, p);
            row = min(row, st.rows - 1);
            const int bb = first && a.nb > 1 ? (int)((unsigned)row * a.mag_s >> 16) : 0;
            if constexpr (MODE == WHOLE_LAST) {
                const T* src = group + row * a.C + min(p * EP, a.C - EP);
                if constexpr (DT == 0) v[i] = __builtin_bit_cast(az_i4, *(const az_f4_u*)src);
                else v[i] = __builtin_bit_cast(az_i4, *(const az_s8_u*)src);
            } else {
                const int at = first ? bb * (a.C - 1) * a.S + row : row * a.C, cs = anew_s(first ? a.S : 1);
                T e[EP];
                #pragma unroll
                for (int j = 0; j < EP; ++j) e[j] = (group + min(p * EP + j, a.C - 1) * cs)[at];
                v[i] = *(az_i4*)e;
            }
        }
    }
    // Rows beyond the step are zero; channels beyond C were zeroed when the kernel began and stay so.
    __device__ __forceinline__ void store(const PolicyDev& a, const Step& st, void* hl, int tid) const {
        constexpr int EP = AzElem<DT>::EP;
        typedef typename AzElem<DT>::T T;
        #pragma unroll
        for (int i = 0; i < NP; ++i) {
            int row, p;
            place(i, tid, row, p);
            const az_i4 x = row < st.rows ? v[i] : az_i4{0, 0, 0, 0};
            T* dst = (T*)hl + row * LDC + p * EP;
            if (p * EP + EP <= a.C) *(az_i4*)dst = x;
            else if (MODE == ANY) {
                T e[EP];
                *(az_i4*)e = x;
                #pragma unroll
                for (int j = 0; j < EP; ++j) if (p * EP + j < a.C) dst[j] = e[j];
            }
        }
    }
};

// The sparse targets of 16 rows (tile rt of the step) and planes o0 .. o0 + n - 1 into t [16][LD], cleared before: one
// wave, the entries in their order (an LDS add takes a wave's lanes in theirs), so an action that is named more than once
// is summed in one order.
// key0, val0: the lane's entry of the step's first 64 (e0 ..).
template <int LD> __device__ __forceinline__ void scatter_targets(const PolicyDev& a, const BoardLds& l, float* t, const Step& st, int rt, int e0, int e1, int key0, float val0, int lane,
                                                                  int o0 = 0, int n = 128) {
    const int row0 = st.cell0 + rt * 16;
    const auto put = [&](int key, float v) __attribute__((always_inline)) {
        const int o = (key & 255) - o0, row = (key >> 8) - row0;
        if (key >= 0 && (unsigned)o < (unsigned)n && (unsigned)row < 16u) __hip_atomic_fetch_add(t + row * LD + o, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    };
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (l.listed) {
        put(key0, val0);
        for (int e = e0 + 64 + lane; e < e1; e += 64) put(l.key[e], l.val[e]);
    } else
        for (int e = lane; e < min(a.nb, a.B - st.b0) * a.cap; e += 64) {
            float v = 0.f;
            const int key = entry_at(a, st.b0, e, v);
            put(key, v);
        }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Gradients.  Eight waves.  A step: dz of 64 rows (16 rows and half of the planes a wave), then its product with w (32
// rows and a quarter of the channels a wave) and its product with the features (half of the planes and a quarter of the
// channels a wave, kept in registers over all of a workgroup's steps).  16-bit features: dz goes to LDS as hi + lo of the
// type, and both feed both products: where planes cancel, hi alone (half a step of the type in each term) was off by up to a
// third of an element of dh, and made its error 1.4 times its own rounding on the whole.  bf16: hi + lo are 16 bits, which shows
// in dw of small batches (an fp32 sum over all rows: up to 5e-6 of it against 1e-7 in fp32); a third part takes hi's place
// once that has been read.
// (16-bit features of up to 128 channels and 96 planes have a kernel of their own below for all but the smallest batches.)
// fp32: bound by the matrix instructions, 32 cycles for the 16 x 16 x 4: 256 boards of 20 x 20, 256 channels, 91 planes
// 222 us, 65 TFLOP/s (three products: 93 us at the rate of a large one; the matrix units work for half of the time).  256 channels leave no registers to ask for the next
// step's features early: kept in flight they went to scratch memory and back (367 us).
template <int DT, int OT, int CB, int MODE> __global__ void __launch_bounds__(NT, 2) az_policy_grad_kernel(PolicyDev a) {
    typedef Lay<DT, OT, CB> L;
    typedef typename AzElem<DT>::T T;
    constexpr int NP = CB * 128 / L::EP * ROWS / NT, OTH = (OT + 1) / 2, KO = L::OP / L::KS, KT = CB * 128 / L::KS;
    constexpr int OG = OT > 1 ? 2 : 1, CG = 8 / OG, OTN = OT / OG, CTN = CB * 8 / CG;   // dw: groups of planes and channels, tiles of a wave
    constexpr bool WLDS = w_in_lds<DT, OT, CB>(), THIRD = DT == 2;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    constexpr int Cp = L::CP, ldc = L::LDC;
    const Smem<DT, OT, CB, 1, WLDS> m(smem, a, L::z_bytes);
    T* zhi = (T*)m.t;
    T* zlo = zhi + ROWS * L::LDO;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, q = lane >> 4, rt = wave & 3, half = wave >> 2;
    const int s_lo = (int)((long long)blockIdx.x * a.steps / gridDim.x), s_hi = (int)((long long)(blockIdx.x + 1) * a.steps / gridDim.x);
    const int og = OG == 2 ? wave & 1 : 0, cg = OG == 2 ? wave >> 1 : wave, pair = wave & 1, cq = wave >> 1;
    az_f4 dw[CTN][OTN];
    #pragma unroll
    for (int i = 0; i < CTN; ++i)
        #pragma unroll
        for (int j = 0; j < OTN; ++j) dw[i][j] = az_f4{0.f, 0.f, 0.f, 0.f};
    az_f4 db[OTH];
    #pragma unroll
    for (int j = 0; j < OTH; ++j) db[j] = az_f4{0.f, 0.f, 0.f, 0.f};
    // fp32, more than 128 channels: a step's features are 32 registers a thread that the products need; they are asked for
    // when the step before is done (on their way earlier they went through scratch memory, a load at a time)
    constexpr bool EARLY = !(DT == 0 && CB == 2);
    Step st(a, s_lo);
    Feat<DT, NP, MODE> f;
    f.load(a, st, tid);
    for (int o = tid; o < OT * 16; o += NT) m.bias[o] = o < a.O ? az_load<DT>(a.bias, o) : 0.f;
    init_words(a, m.b, tid);
    if constexpr (WLDS) stage_w<DT, OT, CB>(a, m.w, tid);
    if (a.C < Cp) for (int i = tid; i < ROWS * ldc; i += NT) ((T*)m.h)[i] = (T)0.f;
    // fp16: dz is r_b (a mean over the batch: 1 / B) times probabilities that may be 1e-5, below what fp16 resolves.  The
    // workgroup's dz carry a power of two that puts the largest of its boards' |r_b| sum |t|, which no dz exceeds, at 2^9 .. 2^10;
    // it comes off the fp32 sums again.  (One power for all: dw sums over them.  A board 2^15 below the largest still has the
    // precision of its gradients' own rounding.)
    float up = 1.f, down = 1.f;
    if constexpr (DT == 1) {
        const Step last(a, s_hi - 1);
        const int b1 = min(last.b0 + a.nb, a.B);
        float mx = 0.f;
        for (int b = st.b0 + tid; b < b1; b += NT) mx = fmaxf(mx, fabsf(a.scale * (a.row_scale ? a.row_scale[b] : 1.f) * a.stats[b][3]));
        mx = wave_max(mx);
        if (lane == 0) m.t[wave] = mx;
        __syncthreads();
        for (int w = 0; w < 8; ++w) mx = fmaxf(mx, m.t[w]);
        if (mx > 0.f && mx < INFINITY) {
            const int e = min(max(10 - (ilogbf(mx) + 1), -100), 100);
            up = ldexpf(1.f, e);
            down = ldexpf(1.f, -e);
        }
    }
    __syncthreads();
    T* h = (T*)m.h;
    f.store(a, st, h, tid);
    stage_boards<true>(a, m.b, st.b0, tid);                          // (ends in a barrier)
    // dense targets of a step, on their way during the step before, ahead of the features (loads return in order)
    az_f4 tv[OTH];
    const auto targets = [&](const PolicyDev& a, const Step& st) __attribute__((always_inline)) {
        const int row = min(rt * 16 + (lane & 15), st.rows - 1), bb = a.nb > 1 ? (int)((unsigned)row * a.mag_s >> 16) : 0, s = st.cell0 + row - bb * a.S;
        const float* dense = a.dense + (size_t)st.b0 * a.O * a.S;
        const int at = (bb * a.O + half * OTH * 16 + q * 4) * a.S + s, last = ((bb + 1) * a.O - 1) * a.S + s;
        #pragma unroll
        for (int j = 0; j < OTH; ++j)
            #pragma unroll
            for (int i = 0; i < 4; ++i) tv[j][i] = dense[min(at + (j * 16 + i) * a.S, last)];   // (dropped where no action stands for it)
    };
    if (!a.counts) targets(a, st);
    Step nx = st;
    if (s_lo + 1 < s_hi) { nx.next(a); if (EARLY) f.load(a, nx, tid); }
    #pragma unroll 1
    for (int it = s_lo; it < s_hi; ++it) {
        const PolicyDev a = arguments();
        // dz of the step
        const int rl = rt * 16 + (lane & 15);
        const bool live = rl < st.rows;
        const int bb = live && a.nb > 1 ? (int)((unsigned)rl * a.mag_s >> 16) : 0, s = live ? st.cell0 + rl - bb * a.S : 0, y = (int)((unsigned)s * a.mag_n >> 16);
        const unsigned bit = live ? 1u << (s - y * a.N) : 0u;
        const unsigned* words = m.b.words + (bb * a.N + y) * (OT * 16) + half * OTH * 16 + q * 4;
        const az_f4 bst = m.b.stat[bb];
        const float rs = up * bst[2];
        if (a.counts) {
            float* t = m.t + rt * 16 * L::LDT;                   // where dz will lie: the waves clear and read it together
            for (int i = tid; i < ROWS * L::LDT / 4; i += NT) ((az_f4*)m.t)[i] = az_f4{0.f, 0.f, 0.f, 0.f};
            __syncthreads();
            const int e0 = m.b.listed ? m.b.start[st.blk] : 0, e1 = m.b.listed ? m.b.start[st.blk + 1] : 0;
            const bool first = e0 + lane < e1;
            scatter_targets<L::LDT>(a, m.b, t + half * OTH * 16, st, rt, e0, e1, first ? m.b.key[e0 + lane] : -1, first ? m.b.val[e0 + lane] : 0.f, lane, half * OTH * 16, OTH * 16);
            #pragma unroll
            for (int j = 0; j < OTH; ++j) tv[j] = half * OTH + j < OT ? *(const az_f4*)(t + (lane & 15) * L::LDT + (half * OTH + j) * 16 + q * 4) : az_f4{0.f, 0.f, 0.f, 0.f};
            __syncthreads();
        }
        az_f4 acc[OTH];
        #pragma unroll
        for (int j = 0; j < OTH; ++j) acc[j] = *(const az_f4*)(m.bias + min(half * OTH + j, OT - 1) * 16 + q * 4);
        const auto step = [&](int k, const az_i4* w) __attribute__((always_inline)) {
            const az_i4 hb = az_row_frag<DT>(h, ldc, rt * 16, k * L::KS, lane);
            #pragma unroll
            for (int j = 0; j < OTH; ++j) acc[j] = az_mma<DT>(w[j], hb, acc[j]);
        };
        const auto fetch = [&](int k, az_i4* w) __attribute__((always_inline)) {
            #pragma unroll
            for (int j = 0; j < OTH; ++j) {
                const int ot = min(half * OTH + j, OT - 1);
                if constexpr (WLDS) w[j] = az_row_frag<DT>(m.w, L::LDW, ot * 16, k * L::KS, lane);
                else w[j] = az_row_frag<DT>(a.wpad, Cp, ot * 16, k * L::KS, lane);
            }
        };
        __builtin_amdgcn_sched_barrier(0);                           // (phases apart: mixed, they want more registers than there are)
        product<KT, L::KS, OTH, !WLDS>(a.C, fetch, step);
        __builtin_amdgcn_sched_barrier(0);
        const float rp = up * bst[1], mz = bst[0];
        // one plane and no target outside the allowed actions: the bias moves every logit alike, its gradient is zero (or NaN
        // with all of the board's)
        const bool bias_counts = OT > 1 || a.O > 1 || bst[3] != 0.f;
        az_s4 rest[THIRD ? OTH : 1];
        #pragma unroll
        for (int j = 0; j < OTH; ++j) {
            const int ot = half * OTH + j;
            if (ot * 16 >= L::OP) continue;
            az_f4 dz = {0.f, 0.f, 0.f, 0.f};
            if (ot < OT) {
                const az_i4 w = *(const az_i4*)(words + j * 16);
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float v = __builtin_fmaf(rp, __builtin_amdgcn_exp2f((acc[j][i] - mz) * LOG2E), -rs * tv[j][i]);
                    dz[i] = (unsigned)w[i] & bit ? v : 0.f;
                }
            }
            if (bias_counts) db[j] += dz;
            if constexpr (DT == 0) *(az_f4*)((float*)zhi + rl * L::LDO + ot * 16 + q * 4) = dz;
            else {
                az_s4 hi, lo;
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    short x, y, z;
                    if constexpr (THIRD) { az_split<DT>(dz[i], x, y, z); rest[j][i] = z; }
                    else az_split<DT>(dz[i], x, y);
                    hi[i] = x;
                    lo[i] = y;
                }
                *(az_s4*)((short*)zhi + rl * L::LDO + ot * 16 + q * 4) = hi;
                *(az_s4*)((short*)zlo + rl * L::LDO + ot * 16 + q * 4) = lo;
            }
        }
        __syncthreads();
        Step after = nx;
        if (it + 2 < s_hi) after.next(a);
        if (!a.counts && it + 1 < s_hi) targets(a, nx);
        // dh: rows of a tile are channels, columns are cells
        {
            // (fp32: dz is read again for every tile of channels -- the LDS port is idle behind the fp32 matrix instructions,
            // and the fragments of both row tiles would take 48 registers; so it is where 16 bits' 64 registers do not fit
            // beside the largest dw)
            constexpr bool KEEP = DT != 0 && !(OT == 8 && CB == 2);
            constexpr int PARTS = DT == 0 ? 1 : 2;
            az_i4 zf[2][KEEP ? KO : 1][PARTS];                       // [row tile][step][hi, lo]
            const auto dz_frag = [&](int e, int k, int p) __attribute__((always_inline)) { return az_row_frag<DT>(p ? zlo : zhi, L::LDO, (pair * 2 + e) * 16, k * L::KS, lane); };
            if constexpr (KEEP) {
                #pragma unroll
                for (int k = 0; k < KO; ++k)
                    #pragma unroll
                    for (int e = 0; e < 2; ++e)
                        #pragma unroll
                        for (int p = 0; p < PARTS; ++p) zf[e][k][p] = dz_frag(e, k, p);
            }
            #pragma unroll 1
            for (int j = 0; j < CB * 2; ++j) {
                const int ct = cq + 4 * j;
                if (ct * 16 >= a.C) continue;
                az_f4 d[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
                #pragma unroll
                for (int k = 0; k < KO; ++k) {
                    az_i4 wa;
                    if constexpr (WLDS) wa = az_col_frag<DT>(m.w, L::LDW, k * L::KS, ct * 16, lane);
                    else wa = az_row_frag<DT>(a.wpadt, L::OP, ct * 16, k * L::KS, lane);
                    #pragma unroll
                    for (int e = 0; e < 2; ++e)
                        #pragma unroll
                        for (int p = 0; p < PARTS; ++p) d[e] = az_mma<DT>(wa, KEEP ? zf[e][KEEP ? k : 0][p] : dz_frag(e, k, p), d[e]);
                }
                const int c = ct * 16 + q * 4;
                #pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int row = (pair * 2 + e) * 16 + (lane & 15);
                    if (row >= st.rows || c >= a.C) continue;
                    if constexpr (DT == 1) d[e] *= down;
                    if (MODE == WHOLE_LAST || (MODE == ANY && !a.nchw)) {
                        T* dst = (T*)a.dh + ((size_t)st.b0 * a.S + st.cell0) * a.C + (row * a.C + c);
                        if (MODE == WHOLE_LAST || c + 4 <= a.C) {
                            if constexpr (DT == 0) *(az_f4_u*)dst = d[e];
                            else *(az_s4_u*)dst = az_s4{az_to16<DT>(d[e][0]), az_to16<DT>(d[e][1]), az_to16<DT>(d[e][2]), az_to16<DT>(d[e][3])};
                        } else for (int i = 0; i < 4; ++i) if (c + i < a.C) az_store<DT>(dst, i, d[e][i]);
                    } else {
                        const int b2 = a.nb > 1 ? (int)((unsigned)row * a.mag_s >> 16) : 0, s2 = st.cell0 + row - b2 * a.S;
                        T* dst = (T*)a.dh + (size_t)st.b0 * a.C * a.S + ((b2 * a.C + c) * a.S + s2);
                        for (int i = 0; i < 4; ++i) if (MODE == WHOLE_FIRST || c + i < a.C) az_store<DT>(dst, (size_t)i * a.S, d[e][i]);
                    }
                }
            }
        }
        // dw: rows of a tile are planes, columns are channels, the contraction runs over the step's rows (rows beyond the
        // step have dz = 0 and features of 0)
        const auto times_features = [&](auto parts) __attribute__((always_inline)) {
            constexpr int P = decltype(parts)::value;
            #pragma unroll
            for (int k = 0; k < ROWS; k += L::KS) {
                if (k >= st.rows) break;
                __builtin_amdgcn_sched_barrier(0);
                az_i4 zf[OTN][P];
                #pragma unroll
                for (int j = 0; j < OTN; ++j) {
                    zf[j][0] = az_col_frag<DT, true>(zhi, L::LDO, k, (og * OTN + j) * 16, lane);
                    if constexpr (P == 2) zf[j][1] = az_col_frag<DT, true>(zlo, L::LDO, k, (og * OTN + j) * 16, lane);
                }
                #pragma unroll
                for (int i = 0; i < CTN; ++i) {
                    const int ct = cg + CG * i;
                    if (ct * 16 >= a.C) continue;
                    const az_i4 hb = az_col_frag<DT, true>(h, ldc, k, ct * 16, lane);
                    #pragma unroll
                    for (int j = 0; j < OTN; ++j)
                        #pragma unroll
                        for (int p = 0; p < P; ++p) dw[i][j] = az_mma<DT>(zf[j][p], hb, dw[i][j]);
                }
            }
        };
        times_features(std::integral_constant<int, DT == 0 ? 1 : 2>{});
        if constexpr (THIRD) {
            __syncthreads();                                         // hi has been read
            #pragma unroll
            for (int j = 0; j < OTH; ++j)
                if ((half * OTH + j) * 16 < L::OP) *(az_s4*)((short*)zhi + rl * L::LDO + (half * OTH + j) * 16 + q * 4) = rest[j];
            __syncthreads();
            times_features(std::integral_constant<int, 1>{});
        }
        __syncthreads();                                             // everything of this step has been read
        if (it + 1 < s_hi) {
            if (!EARLY) f.load(a, nx, tid);
            f.store(a, nx, h, tid);
            if (EARLY && it + 2 < s_hi) f.load(a, after, tid);
            if (nx.b0 == st.b0) __syncthreads();                     // (else the boards' staging ends in one)
        }
        if (it + 1 < s_hi && nx.b0 != st.b0) stage_boards<true>(a, m.b, nx.b0, tid);
        st = nx;
        nx = after;
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
    float* red = m.t;                                                // [4][OT * 16]
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

// Gradients, 16-bit features of up to 128 channels and 96 planes.  Four waves make dz of step t (a row tile each, all planes: mostly
// vector instructions) while the other four multiply dz of step t - 1 both ways (mostly matrix instructions), one of
// either kind on each SIMD, one barrier a step; each kind holds its shares of w in registers.  Done by the same waves one
// after the other, neither the vector nor the matrix pipes nor the LDS port were busy half of the time.  LDS: features of
// three steps, dz (hi and lo) of two, the sparse targets of each row tile.
// 2048 boards of 20 x 20, 128 channels, 91 planes bf16: 200 us, 285 TFLOP/s of useful products (the parts of dz counted
// once), 2.1 TB/s of features and their gradients (86 us of copying); what bounds it is the step's chain of logits, exponentials,
// LDS and products between two barriers with one workgroup a CU (vector units 38 % of the time, matrix units 28 %; LDS bank
// conflicts 13 %).  hi alone for dh and two parts for dw took 158.  4096 boards of 15 x 15, one plane: 92 us, 5.1 TB/s: memory.
template <int DT, int OT> struct PairCfg {
    typedef Lay<DT, OT, 1> L;
    static constexpr int LDP = OT * 16 + 4;
    // bf16: a third part of dz for dw, as in az_policy_grad_kernel.  Its room for 96 planes is that of the sparse targets' tiles:
    // those lie in the rows that the wave's dz is about to take, and are all read before.
    static constexpr bool THIRD = DT == 2, ALIAS = THIRD && OT == 6;
    // A row of dz: its parts side by side, PW planes each, rows an odd multiple of 32 bytes apart (az_col_frag).  Up to 16 planes:
    // hi and lo are one step of the contraction over planes, against w's planes twice.
    static constexpr int PW = OT * 16, LDZ = OT == 1 ? 48 : (THIRD ? 3 : 2) * PW + 16;
    static constexpr size_t own = (size_t)16 * LDP * 4, z = (size_t)ROWS * LDZ * 2;    // a row tile's targets; a step's dz
    static_assert(!ALIAS || own <= (size_t)16 * LDZ * 2, "a tile of targets lies in 16 rows of dz");
    static __host__ __device__ size_t zb(const PolicyDev& a) { return 2 * z + (a.counts && !ALIAS ? 4 * own : 0); }
};
// az_col_frag of 16 columns that are not neighbours: four from n0, four from n0 + 8, ...  TWICE: 16 rows, and the same again.
template <bool TWICE> __device__ __forceinline__ az_i4 pair_col_frag(const void* m, int ld, int k0, int n0, int lane) {
    typedef __attribute__((address_space(3))) az_s4* lds_s4;
    const short* p = (const short*)m + (k0 + 8 * (lane >> 4 & (TWICE ? 1 : 3)) + ((lane & 15) >> 2)) * ld + n0 + (lane & 3) * 8;
    const az_s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)p);
    const az_s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(p + 4 * ld));
    return __builtin_bit_cast(az_i4, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

template <int DT, int OT, int MODE> __global__ void __launch_bounds__(NT, OT == 1 ? 4 : 2) az_policy_grad16_kernel(PolicyDev a) {
    typedef Lay<DT, OT, 1> L;
    typedef PairCfg<DT, OT> G;
    typedef typename AzElem<DT>::T T;
    constexpr int KT = 128 / L::KS, KO = L::OP / L::KS, ldc = L::LDC;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const Smem<DT, OT, 1, 3, false> m(smem, a, G::zb(a));
    T* const hbuf = (T*)m.h;
    T* const zbuf = (T*)m.t;                                         // [2][ROWS][LDZ]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, q = lane >> 4;
    const int s_lo = (int)((long long)blockIdx.x * a.steps / gridDim.x), steps = (int)((long long)(blockIdx.x + 1) * a.steps / gridDim.x) - s_lo;
    Step st(a, s_lo);
    for (int o = tid; o < OT * 16; o += NT) m.bias[o] = o < a.O ? az_load<DT>(a.bias, o) : 0.f;
    init_words(a, m.b, tid);
    // fp16: dz is r_b (a mean over the batch: 1 / B) times probabilities that may be 1e-5, below what fp16 resolves.  The
    // workgroup's dz carry a power of two that puts the largest of its boards' |r_b| sum |t|, which no dz exceeds, at 2^9 .. 2^10;
    // it comes off the fp32 sums again.
    float up = 1.f, down = 1.f;
    if constexpr (DT == 1) {
        const Step last(a, s_lo + steps - 1);
        const int b1 = min(last.b0 + a.nb, a.B);
        float mx = 0.f;
        for (int b = st.b0 + tid; b < b1; b += NT) mx = fmaxf(mx, fabsf(a.scale * (a.row_scale ? a.row_scale[b] : 1.f) * a.stats[b][3]));
        mx = wave_max(mx);
        if (lane == 0) m.t[wave] = mx;
        __syncthreads();
        for (int w = 0; w < 8; ++w) mx = fmaxf(mx, m.t[w]);
        if (mx > 0.f && mx < INFINITY) {
            const int e = min(max(10 - (ilogbf(mx) + 1), -100), 100);
            up = ldexpf(1.f, e);
            down = ldexpf(1.f, -e);
        }
    }
    static_assert(L::w_bytes <= 3 * L::h_bytes, "w passes through the features' room");
    stage_w<DT, OT, 1>(a, m.h, tid);
    __syncthreads();
    float* const out = a.partial + (size_t)blockIdx.x * ((size_t)a.O * a.C + a.O);
    BoardQueue boards;
    if (wave < 4) {
        az_i4 wr[OT][KT];
        #pragma unroll
        for (int j = 0; j < OT; ++j)
            #pragma unroll
            for (int k = 0; k < KT; ++k) wr[j][k] = az_row_frag<DT>(m.h, L::LDW, j * 16, k * L::KS, lane);
        az_f4 db[OT];
        #pragma unroll
        for (int j = 0; j < OT; ++j) db[j] = az_f4{0.f, 0.f, 0.f, 0.f};
        __syncthreads();                                             // w has been read
        if (a.C < L::CP) for (int i = tid; i < 3 * ROWS * ldc; i += NT / 2) hbuf[i] = (T)0.f;
        __syncthreads();
        boards.first(a, m.b, st.b0, tid);
        float* const apart = (float*)((unsigned char*)m.t + 2 * G::z + wave * G::own);
        const int rl = wave * 16 + (lane & 15);
        const auto clear_own = [&](float* own) __attribute__((always_inline)) {
            #pragma unroll
            for (int i = 0; i < (int)(G::own / 16 + 63) / 64; ++i)
                if (i * 64 + lane < (int)(G::own / 16)) ((az_f4*)own)[i * 64 + lane] = az_f4{0.f, 0.f, 0.f, 0.f};
        };
        if (a.counts && !G::ALIAS) clear_own(apart);
        // dense targets of a step: asked for during the step before, ahead of the features (loads return in order)
        az_f4 tv[OT] = {};
        const auto targets = [&](const PolicyDev& a, const Step& st) __attribute__((always_inline)) {
            const int row = min(rl, st.rows - 1), bb = a.nb > 1 ? (int)((unsigned)row * a.mag_s >> 16) : 0, s = st.cell0 + row - bb * a.S;
            const float* dense = a.dense + (size_t)st.b0 * a.O * a.S;
            const int at = (bb * a.O + q * 4) * a.S + s, last = ((bb + 1) * a.O - 1) * a.S + s;
            #pragma unroll
            for (int j = 0; j < OT; ++j)
                #pragma unroll
                for (int i = 0; i < 4; ++i) { const float v = dense[min(at + (j * 16 + i) * a.S, last)]; tv[j][i] = j * 16 + q * 4 + i < a.O ? v : 0.f; }
        };
        if (!a.counts) targets(a, st);
        Step nx = st;
        if (steps > 1) nx.next(a);
        #pragma unroll 1
        for (int t = 0; t < steps; ++t) {
            const PolicyDev a = arguments();
            if (t && st.blk == 0) boards.next(a, m.b, st.b0, tid);
            const int e0 = m.b.listed ? m.b.start[st.blk] : 0, e1 = m.b.listed ? m.b.start[st.blk + 1] : 0;
            int key0 = -1;
            float val0 = 0.f;
            if (e0 + lane < e1) { key0 = m.b.key[e0 + lane]; val0 = m.b.val[e0 + lane]; }
            const T* h = hbuf + t % 3 * ROWS * ldc;
            short* const dzr = (short*)zbuf + (t & 1) * (G::z / 2) + rl * G::LDZ;
            float* const own = G::ALIAS ? (float*)((short*)zbuf + (t & 1) * (G::z / 2) + wave * 16 * G::LDZ) : apart;
            const bool live = rl < st.rows;
            const int bb = live && a.nb > 1 ? (int)((unsigned)rl * a.mag_s >> 16) : 0, s = live ? st.cell0 + rl - bb * a.S : 0, y = (int)((unsigned)s * a.mag_n >> 16);
            const unsigned bit = live ? 1u << (s - y * a.N) : 0u;
            const unsigned* words = m.b.words + (bb * a.N + y) * (OT * 16) + q * 4;
            const az_f4 bst = m.b.stat[bb];
            if (a.counts) {
                if (G::ALIAS) clear_own(own);
                scatter_targets<G::LDP>(a, m.b, own, st, wave, e0, e1, key0, val0, lane);
                if (G::ALIAS) {
                    #pragma unroll
                    for (int j = 0; j < OT; ++j) tv[j] = *(const az_f4*)(own + (lane & 15) * G::LDP + j * 16 + q * 4);
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    __builtin_amdgcn_wave_barrier();
                }
            }
            // a row behind the board's last has the biases as its logits, which may lie far above the board's largest: its maximum
            // is taken as infinite, its exponentials are 0
            const float rs = live ? up * bst[2] : 0.f, rp = live ? up * bst[1] : 0.f, mz = live ? bst[0] : INFINITY;
            // one plane and no target outside the allowed actions: the bias moves every logit alike, its gradient is zero (or NaN
            // with all of the board's)
            const bool bias_counts = OT > 1 || a.O > 1 || bst[3] != 0.f;
            constexpr int OH = OT > 2 ? OT / 2 : OT;                 // planes in two halves: fewer registers
            #pragma unroll
            for (int j0 = 0; j0 < OT; j0 += OH) {
                az_f4 acc[OH];
                #pragma unroll
                for (int j = 0; j < OH; ++j) acc[j] = *(const az_f4*)(m.bias + (j0 + j) * 16 + q * 4);
                #pragma unroll
                for (int k = 0; k < KT; ++k) {
                    const az_i4 hb = az_row_frag<DT>(h, ldc, wave * 16, k * L::KS, lane);
                    #pragma unroll
                    for (int j = 0; j < OH; ++j) acc[j] = az_mma<DT>(wr[j0 + j][k], hb, acc[j]);
                }
                if (a.counts && !G::ALIAS) {
                    #pragma unroll
                    for (int j = 0; j < OH; ++j) tv[j0 + j] = *(const az_f4*)(own + (lane & 15) * G::LDP + (j0 + j) * 16 + q * 4);
                }
                #pragma unroll
                for (int j = 0; j < OH; ++j) {
                    const int o = (j0 + j) * 16 + q * 4;
                    az_f4 dz;
                    #pragma unroll
                    for (int i = 0; i < 4; ++i) dz[i] = __builtin_fmaf(rp, __builtin_amdgcn_exp2f((acc[j][i] - mz) * LOG2E), -rs * tv[j0 + j][i]);
                    if (a.legal) {
                        const az_i4 w = *(const az_i4*)(words + (j0 + j) * 16);
                        #pragma unroll
                        for (int i = 0; i < 4; ++i) dz[i] = (unsigned)w[i] & bit ? dz[i] : 0.f;
                    } else if (j0 + j >= (OT > 2 ? OT - 2 : OT - 1) && (j0 + j) * 16 + 16 > a.O) {
                        // planes there are not: infinite features times weights of 0 (only the last tiles may have them)
                        #pragma unroll
                        for (int i = 0; i < 4; ++i) dz[i] = o + i < a.O ? dz[i] : 0.f;
                    }
                    if (bias_counts) db[j0 + j] += dz;
                    az_s4 hi, lo, rest;
                    #pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        short x, y, z;
                        if constexpr (G::THIRD) { az_split<DT>(dz[i], x, y, z); rest[i] = z; }
                        else az_split<DT>(dz[i], x, y);
                        hi[i] = x;
                        lo[i] = y;
                    }
                    *(az_s4*)(dzr + o) = hi;
                    *(az_s4*)(dzr + G::PW + o) = lo;
                    if constexpr (G::THIRD) *(az_s4*)(dzr + 2 * G::PW + o) = rest;
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (a.counts && !G::ALIAS) clear_own(apart);
            if (!a.counts && t + 1 < steps) targets(a, nx);
            st = nx;
            if (t + 2 < steps) nx.next(a);
            __syncthreads();
        }
        float* const r4 = (float*)(hbuf + steps % 3 * ROWS * ldc);   // (the other waves still read the features of step steps - 1)
        #pragma unroll
        for (int j = 0; j < OT; ++j)
            #pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v = db[j][i];
                for (int d = 1; d < 16; d <<= 1) v += __shfl_xor(v, d, 64);
                if ((lane & 15) == 0) r4[wave * OT * 16 + j * 16 + q * 4 + i] = v;
            }
        __syncthreads();
        for (int o = tid; o < a.O; o += NT / 2) out[(size_t)a.O * a.C + o] = ((r4[o] + r4[OT * 16 + o]) + (r4[2 * OT * 16 + o] + r4[3 * OT * 16 + o])) * down;
    } else {
        const int cq = wave - 4, tb = tid - NT / 2;                  // channels 32 cq .. + 31
        az_i4 wc[2][KO];
        #pragma unroll
        for (int j = 0; j < 2; ++j)
            #pragma unroll
            for (int k = 0; k < KO; ++k) wc[j][k] = pair_col_frag<OT == 1>(m.h, L::LDW, k * L::KS, cq * 32 + 4 * j, lane);
        az_f4 dw[2][OT];
        #pragma unroll
        for (int i = 0; i < 2; ++i)
            #pragma unroll
            for (int j = 0; j < OT; ++j) dw[i][j] = az_f4{0.f, 0.f, 0.f, 0.f};
        // features: step t + 1 goes to LDS at the start of interval t (in which dz of step t are made and those of step t - 1
        // multiplied), t + 2 and t + 3 are on their way
        Feat<DT, 4, MODE, 4> f[2];
        Step s0 = st, s1 = st, s2 = st;                              // steps t - 1 .. t + 1; s3: t + 2
        f[0].load(a, st, tb);
        if (steps > 1) { s1.next(a); f[1].load(a, s1, tb); }
        s2 = s1;
        if (steps > 2) s2.next(a);
        __syncthreads();
        __syncthreads();                                             // w has been read, the padding cleared
        f[0].store(a, st, hbuf, tb);
        if (steps > 2) f[0].load(a, s2, tb);
        boards.first(a, m.b, st.b0, tid);
        // interval 0
        if (steps > 1) f[1].store(a, s1, hbuf + ROWS * ldc, tb);
        Step s3 = s2;
        if (steps > 3) { s3.next(a); f[1].load(a, s3, tb); }
        __syncthreads();                                             // dz of step 0
        const auto interval = [&](int t, Feat<DT, 4, MODE, 4>& f) __attribute__((always_inline)) {   // multiplies step t; interval t + 1
            const PolicyDev a = arguments();
            const Step st = s0;
            if (t + 1 < steps && s1.blk == 0) boards.next(a, m.b, s1.b0, tid);   // (with the other waves, ahead of their step t + 1)
            if (t + 2 < steps) f.store(a, s2, hbuf + (t + 2) % 3 * ROWS * ldc, tb);
            s0 = s1; s1 = s2; s2 = s3;
            if (t + 4 < steps) { s3.next(a); f.load(a, s3, tb); }
            const T* h = hbuf + t % 3 * ROWS * ldc;
            const T* const zt = zbuf + (t & 1) * (G::z / 2);
            // dh: rows of a tile are channels, columns are cells
            #pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (e * 16 >= st.rows) break;
                az_f4 d[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
                #pragma unroll
                for (int k = 0; k < KO; ++k) {
                    #pragma unroll
                    for (int part = 0; part < (OT == 1 ? 1 : 2); ++part) {       // (one plane tile: hi and lo in one)
                        const az_i4 zf = az_row_frag<DT>(zt, G::LDZ, e * 16, part * G::PW + k * L::KS, lane);
                        d[0] = az_mma<DT>(wc[0][k], zf, d[0]);
                        d[1] = az_mma<DT>(wc[1][k], zf, d[1]);
                    }
                }
                const int row = e * 16 + (lane & 15), c = cq * 32 + q * 8;       // the two tiles hold 8 channels of the row in turn
                if (row >= st.rows || c >= a.C) continue;
                if constexpr (DT == 1) { d[0] *= down; d[1] *= down; }
                az_s8 o;
                #pragma unroll
                for (int i = 0; i < 8; ++i) o[i] = az_to16<DT>(d[i >> 2][i & 3]);
                if (MODE == WHOLE_LAST || (MODE == ANY && !a.nchw)) {
                    short* dst = (short*)a.dh + ((size_t)st.b0 * a.S + st.cell0) * a.C + (row * a.C + c);
                    if (MODE == WHOLE_LAST || c + 8 <= a.C) *(az_s8_u*)dst = o;
                    else {
                        #pragma unroll
                        for (int i = 0; i < 8; ++i) if (c + i < a.C) dst[i] = o[i];
                    }
                } else {
                    const int b2 = a.nb > 1 ? (int)((unsigned)row * a.mag_s >> 16) : 0;
                    short* dst = (short*)a.dh + (size_t)st.b0 * a.C * a.S + ((b2 * a.C + c) * a.S + st.cell0 + row - b2 * a.S);
                    #pragma unroll
                    for (int i = 0; i < 8; ++i) if (MODE == WHOLE_FIRST || c + i < a.C) dst[(size_t)i * a.S] = o[i];
                }
            }
            // dw: rows of a tile are planes, columns are channels, the contraction runs over the step's rows (rows beyond the
            // step have dz = 0 and features of 0)
            #pragma unroll
            for (int k = 0; k < ROWS; k += L::KS) {
                if (k >= st.rows) break;
                const az_i4 hb0 = az_col_frag<DT, true>(h, ldc, k, cq * 32, lane), hb1 = az_col_frag<DT, true>(h, ldc, k, cq * 32 + 16, lane);
                #pragma unroll
                for (int j = 0; j < OT; ++j) {
                    const az_i4 z1 = az_col_frag<DT, true>(zt, G::LDZ, k, j * 16, lane), z2 = az_col_frag<DT, true>(zt, G::LDZ, k, G::PW + j * 16, lane);
                    dw[0][j] = az_mma<DT>(z1, hb0, dw[0][j]);
                    dw[1][j] = az_mma<DT>(z1, hb1, dw[1][j]);
                    dw[0][j] = az_mma<DT>(z2, hb0, dw[0][j]);
                    dw[1][j] = az_mma<DT>(z2, hb1, dw[1][j]);
                    if constexpr (G::THIRD) {
                        const az_i4 z3 = az_col_frag<DT, true>(zt, G::LDZ, k, 2 * G::PW + j * 16, lane);
                        dw[0][j] = az_mma<DT>(z3, hb0, dw[0][j]);
                        dw[1][j] = az_mma<DT>(z3, hb1, dw[1][j]);
                    }
                }
            }
            if (t + 1 < steps) __syncthreads();
        };
        #pragma unroll 1
        for (int t = 0; t < steps; t += 2) {
            interval(t, f[0]);
            if (t + 1 < steps) interval(t + 1, f[1]);
        }
        #pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int c = cq * 32 + i * 16 + (lane & 15);
            #pragma unroll
            for (int j = 0; j < OT; ++j)
                #pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int o = j * 16 + q * 4 + e;
                    if (o < a.O && c < a.C) out[(size_t)o * a.C + c] = dw[i][j][e] * down;
                }
        }
        __syncthreads();
    }
}

constexpr size_t LOSS_STATIC = (size_t)4 * ROWS * 16 + MAX_BOARDS * 4;           // az_policy_loss_kernel's `red` and `negative`
template <int DT, int OT, int CB, int MODE> hipError_t launch_products(PolicyDev a, bool grad, int& groups, hipStream_t stream) {
    // az_policy_grad16_kernel: 16-bit features of up to 128 channels and 96 planes (with more, w's shares do not fit the
    // registers), where a workgroup has more than a step.  20 x 20, 91 planes bf16: 2048 boards 287 us a call, with
    // az_policy_grad_kernel 382; 128 boards 47 and 52; at the border, 38 boards (266 steps) 40 and 42.5, 36 (252 steps) 41 and 42;
    // 9 x 9, 3 planes fp16: 140 boards (280 steps) 30 and 29, 77 boards 28 and 27.
    constexpr bool PAIR = DT != 0 && CB == 1 && OT <= 6;
    const bool pair = PAIR && a.steps > CUS;
    const auto bytes = [&]() -> size_t {
        if (!grad) return Smem<DT, OT, CB, 0, w_in_lds<DT, OT, CB>()>::bytes(a, a.counts ? WAVES * LossTile<OT>::bytes : 0) + LOSS_STATIC;
        if constexpr (PAIR) if (pair) return Smem<DT, OT, 1, 3, false>::bytes(a, PairCfg<DT, OT>::zb(a));
        return Smem<DT, OT, CB, 1, w_in_lds<DT, OT, CB>()>::bytes(a, Lay<DT, OT, CB>::z_bytes);
    };
    size_t lds = bytes();
    if (lds > LDS_BYTES) { a.room = 0; lds = bytes(); }              // the longest lists with the largest boards and heads: targets read from memory
    if (lds > LDS_BYTES) return hipErrorInvalidConfiguration;
    const void* fn;
    if (!grad) fn = (const void*)az_policy_loss_kernel<DT, OT, CB, MODE>;
    else fn = (const void*)az_policy_grad_kernel<DT, OT, CB, MODE>;
    if constexpr (PAIR) if (grad && pair) fn = (const void*)az_policy_grad16_kernel<DT, OT, MODE>;
    if (lds > 32 * 1024) {
        const hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    if (!grad) {
        // as many workgroups as the chip holds at once, the boards in even shares
        const int per_cu = loss_waves<DT, OT, CB>() * 4 / WAVES >= 2 && lds * 2 <= LDS_BYTES ? 2 : 1;
        const int work = (a.B + a.nb - 1) / a.nb, room = CUS * per_cu, rounds = (work + room - 1) / room;
        az_policy_loss_kernel<DT, OT, CB, MODE><<<(work + rounds - 1) / rounds, NT, lds - LOSS_STATIC, stream>>>(a, work);
    } else {
        if (lds * 2 > LDS_BYTES && groups > CUS) groups = CUS;       // one workgroup a CU
        if constexpr (PAIR) if (pair) { az_policy_grad16_kernel<DT, OT, MODE><<<groups, NT, lds, stream>>>(a); return hipGetLastError(); }
        az_policy_grad_kernel<DT, OT, CB, MODE><<<groups, NT, lds, stream>>>(a);
    }
    return hipGetLastError();
}
template <int DT, int OT, int CB> hipError_t launch_mode(const PolicyDev& a, bool grad, int& groups, hipStream_t stream) {
    if (a.C % AzElem<DT>::KS) return launch_products<DT, OT, CB, ANY>(a, grad, groups, stream);
    return a.nchw ? launch_products<DT, OT, CB, WHOLE_FIRST>(a, grad, groups, stream) : launch_products<DT, OT, CB, WHOLE_LAST>(a, grad, groups, stream);
}
template <int DT, int OT> hipError_t launch_c(const PolicyDev& a, bool grad, int& groups, hipStream_t stream) {
    return a.C <= 128 ? launch_mode<DT, OT, 1>(a, grad, groups, stream) : launch_mode<DT, OT, 2>(a, grad, groups, stream);
}
template <int DT> hipError_t launch_o(const PolicyDev& a, bool grad, int& groups, hipStream_t stream) {
    if (a.O <= 16) return launch_c<DT, 1>(a, grad, groups, stream);
    if (a.O <= 32) return launch_c<DT, 2>(a, grad, groups, stream);
    if (a.O <= 64) return launch_c<DT, 4>(a, grad, groups, stream);
    if (a.O <= 96) return launch_c<DT, 6>(a, grad, groups, stream);
    return launch_c<DT, 8>(a, grad, groups, stream);
}

}  // namespace
