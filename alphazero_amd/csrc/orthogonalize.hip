// orthogonalize.hip -- an update matrix orthogonalised by Newton-Schulz products, and the optimiser step around it.
//
//   X0 = U / (|U|_F + eps);   X <- a X + (b A + c A^2) X,  A = X X^T,  a number of times;   result s X
//
// The singular vectors stay what they are and every singular value x goes to a x + b x^3 + c x^5.  With X r x k, r <= k
// (a taller matrix is read transposed), every iterate is Q X0 with Q a polynomial of A0 = X0 X0^T, and A, Q and
// P = a + b A + c A^2 all commute and are symmetric:
//   P = a I + b A + c A A,   Q <- Q P,   A <- P A P
// so the long dimension is touched twice, for A0 and for Q X0, and what lies between are r x r products: 4 r^3 k-free
// products a step instead of 2 r^2 k + r^3.  The price is that a singular value is carried as its square: one that is
// small against the largest keeps the absolute precision of A's arithmetic, and the steps enlarge that error as they
// enlarge the value (a^2 each).  So the products run on pairs of fp16 values, s x = hi + lo (22 bits, s a power of two that
// keeps lo out of fp16's subnormals where it matters; three MFMA a product, fp32 sums), and for fp32 results X is formed
// anew after two steps and A from it (16-bit results: after three, make_plan): for matrices whose largest singular value stands for most of the norm three steps
// leave 6 times fp32's error (64 x 225 with 8 strong directions: 6e-6, two steps 1.1e-6, products in fp32 1.1e-6), two steps
// at most fp32's.  fp32 matrix instructions would run at 154 TFLOP/s, three fp16 ones at 1.1 / 3 PFLOP/s.
//
// Measured on an MI355X that copies 4.9 TB/s and multiplies 1.1 PFLOP/s (fp16): 2 x 4096 x 1024 fp32 655 us (eleven
// r x r launches of 25 us, X X^T 75 + 52 + 52 us, Q X 71 + 65 + 65 us; the Gram form's operations are 276 us at the rate of
// a large product); optimiser step of 40 x 256 x 2304 590 us (momentum and norm 65 us at 5.7 TB/s, X X^T 68 + 50 + 50, r x r 11
// launches of 12, Q X 78 + 70 + 92 us, the last with weights read and written).  18 x 128 x 1152 bf16 106 us.
#include "../../include/az_hip.h"
#include "az_learn.h"

#include <cmath>
#include <cstdarg>
#include <cstdio>

namespace {

int ofail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap; va_start(ap, fmt); vsnprintf(buf, sizeof buf, fmt, ap); va_end(ap);
    return az_internal_fail(code, buf);
}

constexpr float SA = 256.f, SQ = 16.f;        // scales of the pairs: A, P and A P (at most about 4), Q (a^5 = 485)
// Contraction of one step of a tile product: 64 halves are a whole 128-byte line of a row; tiles of 128 would then leave
// LDS for one workgroup a CU.
template <int TILE> constexpr int kstep() { return TILE == 64 ? 64 : 32; }
constexpr int MAX_SLICES = 256;               // pieces of a matrix whose squares are summed apart
constexpr int SRC_PAIR = 3;                   // operand kinds: AZ_F32, AZ_F16, AZ_BF16, or pairs

enum { GRAM_WIDE, GRAM_TALL, APPLY_WIDE, APPLY_TALL, SYM };          // what a tile product computes
enum { EPI_PAIR, EPI_PARTIAL, EPI_POLY };                             // what SYM / GRAM leave

struct OrthoDev {
    const void* x;            // operand X: the update
    size_t x_stride;          // elements from matrix to matrix
    int rows, cols, r, k, rp; // as stored; r = min, k = max; rp = r padded to the tile
    int slices;
    const double* sq;         // [n][slices] sums of squares, or null: X is an iterate
    int scale_exp;            // an iterate's power of two
    float eps, a, b, c;
    short *A, *P, *T, *Q, *Q2;// [n][2][rp][rp]: hi plane, lo plane
    float* partial;           // [n][split][rp][rp]
    int split;
    const short* xp;          // an iterate as pairs: [n][2][lines][xld], both sides padded and zero there
    short* xo;                // where the result goes as such pairs (null: the call's own result)
    int xld;
    size_t xplane;
    // result
    void* out;
    size_t out_stride;
    int out_dtype;
    float scale;
    const float* w;           // optimiser step: out = keep * w + scale * X
    size_t w_stride;
    float keep;
};

// |U|_F of matrix z, and the power of two under which its elements are split into pairs: root mean square near 4, but the norm,
// which one element may be most of, at most 2^15 (fp16 ends at 65504; matrices beyond 2^26 elements lose up to 3 of 22 bits to that).
// Every wave by itself, in one order.
__device__ __forceinline__ void norm_of(const OrthoDev& d, int z, int& e, float& back) {
    if (!d.sq) { e = d.scale_exp; back = ldexpf(1.f, -e); return; }
    double s = 0.0;
    for (int i = threadIdx.x & 63; i < d.slices; i += 64) s += d.sq[(size_t)z * d.slices + i];
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    const double norm = sqrt(s);
    e = 0;
    if (norm > 0.0 && norm < 1e300) e = min(max(min(ilogb(sqrt((double)d.r * d.k) / norm) + 2, 14 - ilogb(norm)), -120), 120);
    back = (float)ldexp(1.0 / (norm + (double)d.eps), -e);
}

// sums of squares of a matrix's slices; with mom the update itself: m' = beta m + g, u = nesterov ? g + beta m' : m'.  Four
// elements a thread and load, four loads in flight; what a slice leaves over (and whatever is not there) is dropped.
template <int DT> __device__ __forceinline__ az_f4 load4(const void* p, size_t i) {
    if constexpr (DT == 0) return *(const az_f4_u*)((const float*)p + i);
    else {
        const az_s4 x = *(const az_s4_u*)((const short*)p + i);
        return az_f4{az_from16<DT>(x[0]), az_from16<DT>(x[1]), az_from16<DT>(x[2]), az_from16<DT>(x[3])};
    }
}
template <int DT, bool MOM> __global__ void __launch_bounds__(256) az_ortho_norm_kernel(const void* g, size_t g_stride, int count, int slices, double* sq,
                                                                                     const float* mom, size_t m_stride, float* mom_out, size_t mo_stride, float* u, float beta, int nesterov) {
    __shared__ double red[4];
    const int z = blockIdx.y, sl = blockIdx.x, quads = count / 4;
    const int lo = (int)((long long)quads * sl / slices), hi = (int)((long long)quads * (sl + 1) / slices);
    const size_t go = z * g_stride, mo = z * m_stride, oo = z * mo_stride, uo = (size_t)z * count;
    double s = 0.0;
    const auto one = [&](float v, float m) __attribute__((always_inline)) { return beta * m + v; };
    constexpr int U = 4;
    for (int base = lo + threadIdx.x; base < hi; base += 256 * U) {
        az_f4 v[U], m[U];
        #pragma unroll
        for (int k = 0; k < U; ++k) {
            const size_t i = (size_t)min(base + k * 256, hi - 1) * 4;
            v[k] = load4<DT>(g, go + i);
            if (MOM) m[k] = *(const az_f4_u*)(mom + mo + i);
        }
        #pragma unroll
        for (int k = 0; k < U; ++k) {
            if (base + k * 256 >= hi) break;
            const size_t i = (size_t)(base + k * 256) * 4;
            if (MOM) {
                az_f4 n;
                #pragma unroll
                for (int e = 0; e < 4; ++e) { n[e] = one(v[k][e], m[k][e]); v[k][e] = nesterov ? v[k][e] + beta * n[e] : n[e]; }
                *(az_f4_u*)(mom_out + oo + i) = n;
                *(az_f4_u*)(u + uo + i) = v[k];
            }
            #pragma unroll
            for (int e = 0; e < 4; ++e) s += (double)v[k][e] * v[k][e];
        }
    }
    if (sl == slices - 1 && (int)threadIdx.x < count - quads * 4) {
        const size_t i = (size_t)quads * 4 + threadIdx.x;
        float v = az_load<DT>(g, go + i);
        if (MOM) {
            const float n = one(v, mom[mo + i]);
            v = nesterov ? v + beta * n : n;
            mom_out[oo + i] = n;
            u[uo + i] = v;
        }
        s += (double)v * v;
    }
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) sq[(size_t)z * slices + sl] = (red[0] + red[1]) + (red[2] + red[3]);
}

__device__ __forceinline__ void split(float x, short& hi, short& lo) { az_split<1>(x, hi, lo); }

// One operand of a tile product: TILE lines-or-columns by KSTEP.  ALONG: the contraction runs along a line of memory (LDS
// rows are the tile's rows); otherwise lines are the contraction (LDS rows are its steps, read transposed).  A thread
// carries pieces of 8 elements of a line, as they lie in memory (the loads are unconditional, clamped into the matrix, and
// stay in flight over a step's products), and splits them into hi (and lo) halves on their way to LDS.
template <int TILE, int SRC, bool ALONG> struct Operand {
    static constexpr int KSTEP = kstep<TILE>();
    static constexpr int PARTS = SRC == 0 || SRC == SRC_PAIR ? 2 : 1, RAW = PARTS;
    static constexpr int LD = ALONG ? KSTEP + 8 : TILE + 16;
    static constexpr int LINES = ALONG ? TILE : KSTEP, PER = (ALONG ? KSTEP : TILE) / 8;
    static constexpr int NP = LINES * PER / 256;                     // pieces a thread
    static constexpr int HALVES = LINES * LD;                        // of one part
    az_i4 raw[NP][RAW];
    static __device__ __forceinline__ void place(int i, int tid, int& line, int& pos) { const int w = tid + i * 256; line = w / PER; pos = w % PER * 8; }
    // p (and plo, a pair's lo plane): the matrix; t0, k0: the tile's corner; nlines x npos: the matrix as stored
    __device__ __forceinline__ void load(const void* p, const void* plo, int ld, int t0, int k0, int nlines, int npos, int tid) {
        #pragma unroll
        for (int i = 0; i < NP; ++i) {
            int line, pos;
            place(i, tid, line, pos);
            line += ALONG ? t0 : k0;
            pos += ALONG ? k0 : t0;
            if constexpr (SRC == SRC_PAIR) {
                raw[i][0] = *(const az_i4*)((const short*)p + (size_t)line * ld + pos);
                raw[i][1] = *(const az_i4*)((const short*)plo + (size_t)line * ld + pos);
            } else {
                line = min(line, nlines - 1);
                if (npos >= 8) {
                    // a piece that hangs over the line's end is the line's last 8 elements
                    const size_t at = (size_t)line * ld + min(pos, npos - 8);
                    if constexpr (SRC == 0) {
                        raw[i][0] = __builtin_bit_cast(az_i4, *(const az_f4_u*)((const float*)p + at));
                        raw[i][1] = __builtin_bit_cast(az_i4, *(const az_f4_u*)((const float*)p + at + 4));
                    } else raw[i][0] = __builtin_bit_cast(az_i4, *(const az_s8_u*)((const short*)p + at));
                } else {                                             // short lines: an element a load
                    #pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const size_t at = (size_t)line * ld + min(pos + e, npos - 1);
                        if constexpr (SRC == 0) raw[i][e >> 2][e & 3] = ((const int*)p)[at];
                        else {
                            const int v = ((const unsigned short*)p)[at];
                            raw[i][0][e >> 1] = e & 1 ? raw[i][0][e >> 1] | v << 16 : v;
                        }
                    }
                }
            }
        }
    }
    __device__ __forceinline__ void store(short* s, int t0, int k0, int nlines, int npos, float up, int tid) const {
        #pragma unroll
        for (int i = 0; i < NP; ++i) {
            int line, pos;
            place(i, tid, line, pos);
            short* dst = s + line * LD + pos;
            if constexpr (SRC == SRC_PAIR) {
                *(az_i4*)dst = raw[i][0];
                *(az_i4*)(dst + HALVES) = raw[i][1];
            } else {
                line += ALONG ? t0 : k0;
                pos += ALONG ? k0 : t0;
                az_s8 hi, lo;
                #pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float x;
                    if constexpr (SRC == 0) x = __int_as_float(raw[i][e >> 2][e & 3]);
                    else x = az_from16<SRC>((short)(raw[i][0][e >> 1] >> (e & 1) * 16));
                    x *= up;
                    hi[e] = az_to16<1>(x);
                    lo[e] = SRC == 0 ? az_to16<1>(x - az_from16<1>(hi[e])) : (short)0;
                }
                if (line < nlines && pos + 8 <= npos) {
                    *(az_s8*)dst = hi;
                    if constexpr (PARTS == 2) *(az_s8*)(dst + HALVES) = lo;
                } else {                                             // the matrix's edge: what lies beyond is zero
                    const int first = npos >= 8 ? min(pos, npos - 8) : pos;      // of the piece as loaded
                    #pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (line >= nlines || pos + e >= npos) { dst[e] = 0; if constexpr (PARTS == 2) dst[HALVES + e] = 0; }
                    #pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int at = first + e - pos;
                        if (line < nlines && at >= 0 && pos + at < npos) { dst[at] = hi[e]; if constexpr (PARTS == 2) dst[HALVES + at] = lo[e]; }
                    }
                }
            }
        }
    }
    static __device__ __forceinline__ az_i4 frag(const short* s, int part, int t, int k, int lane) {
        if constexpr (ALONG) return az_row_frag<1>(s + part * HALVES, LD, t, k, lane);
        else return az_col_frag<1>(s + part * HALVES, LD, k, t, lane);
    }
};

// tile (ti, tj) of the lower triangle, ti >= tj, from a running number
__device__ __forceinline__ void lower_tile(int i, int& ti, int& tj) {
    ti = (int)((sqrtf(8.f * i + 1.f) - 1.f) * 0.5f);
    while ((ti + 1) * (ti + 2) / 2 <= i) ++ti;
    while (ti * (ti + 1) / 2 > i) --ti;
    tj = i - ti * (ti + 1) / 2;
}

// entries (nn, m .. m + 3) of a symmetric result as pairs, v at its scale; mirror: and (m .. m + 3, nn)
__device__ __forceinline__ void put_symmetric(const OrthoDev& d, short* res, int z, int m, int nn, bool mirror, az_f4 v) {
    short* hi = res + (size_t)z * 2 * d.rp * d.rp;
    short* lo = hi + (size_t)d.rp * d.rp;
    az_s4 h, l;
    #pragma unroll
    for (int t = 0; t < 4; ++t) { short x, y; split(v[t], x, y); h[t] = x; l[t] = y; }
    *(az_s4*)(hi + (size_t)nn * d.rp + m) = h;
    *(az_s4*)(lo + (size_t)nn * d.rp + m) = l;
    if (mirror)
        #pragma unroll
        for (int t = 0; t < 4; ++t) { hi[(size_t)(m + t) * d.rp + nn] = h[t]; lo[(size_t)(m + t) * d.rp + nn] = l[t]; }
}

// One tile of a product.  Bound by a workgroup's own chain -- loads, LDS, products, barrier: 1.4 us a step of 64 where it
// has its CU to itself, against 0.2 us of matrix instructions.  X X^T and the r x r products take tiles of 64:
// 2 x 4096 x 1024 674 us a call, in tiles of 128 803, 16 x 4096 x 1024 3.6 ms either way, 300 x 128 x 1152 bf16 (five steps a
// stage then) 227 and 241 us.  An r x r product of 2 x 1024 rows 25 us; its operands straight from memory to fragments, without LDS, 39.
// Q X: tiles of 128 where those fill the chip (16 x 4096 x 1024: 3.7 ms a call, in tiles of 64 4.2; 2 x 4096 x 1024 646 and 708 us;
// 40 x 256 x 2304 585 and 609).  By counters the matrix units work for 36 % of Q X in tiles of 128, LDS bank conflicts of the operand
// read by columns take 24 %.
// D[m][n] = sum over the contraction, 4 waves of TILE/2 x TILE/2.  Lane l of a 16 x 16 tile holds rows 4 (l / 16) .. + 3 of
// column l % 16, so M is the side along which the result is contiguous in memory.
//   SYM         M = rows of a symmetric matrix, N = rows of another that commutes with it: their product, lower triangle
//   GRAM_*      M = N = rows of X: lower triangle
//   APPLY_WIDE  M = columns of X, N = rows of Q;   APPLY_TALL  M = rows of Q, N = rows of X as stored (columns of X)
template <int TILE, int DT, int MODE> __global__ void __launch_bounds__(256, 2) az_ortho_product_kernel(OrthoDev d, const short* ma, const short* na, short* res,
                                                                                                 const short* ma2, const short* na2, short* res2, int epi, int n) {                                      // n: tiles of a matrix
    constexpr bool GRAM = MODE == GRAM_WIDE || MODE == GRAM_TALL;
    constexpr int MS = MODE == SYM || MODE == APPLY_TALL ? SRC_PAIR : DT, NS = MODE == SYM || MODE == APPLY_WIDE ? SRC_PAIR : DT;
    constexpr bool MA = !(MODE == GRAM_TALL || MODE == APPLY_WIDE), NA = MODE != GRAM_TALL;
    typedef Operand<TILE, MS, MA> OM;
    typedef Operand<TILE, NS, NA> ON;
    constexpr int KSTEP = kstep<TILE>();
    constexpr int WT = TILE / 2 / 16;                                // 16 x 16 tiles of a wave, each way
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    constexpr int STAGE = OM::PARTS * OM::HALVES + ON::PARTS * ON::HALVES;
    short* lds = (short*)smem;                                       // two stages
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, q = lane >> 4;
    // Workgroups go to the 8 XCDs in turn; each XCD gets a run of tiles, so that the panels that neighbouring tiles (and
    // the next launch's products of the same matrix) read are in its own L2.
    const int total = gridDim.x, run = total / 8, rest = total % 8, xcd = blockIdx.x & 7, at = blockIdx.x >> 3;
    const int tile = xcd * run + min(xcd, rest) + at;
    int z, m0, n0, k_lo = 0, k_hi, sp = 0;
    const size_t plane = (size_t)d.rp * d.rp;
    if constexpr (MODE == SYM || GRAM) {
        int ti, tj;
        z = tile / n;
        lower_tile(tile - z * n, ti, tj);
        m0 = tj * TILE; n0 = ti * TILE;
        if constexpr (GRAM) {
            sp = blockIdx.y;
            const int steps = (d.k + KSTEP - 1) / KSTEP;
            k_lo = steps * sp / d.split * KSTEP;
            k_hi = steps * (sp + 1) / d.split * KSTEP;
        } else {
            if (blockIdx.y) { ma = ma2; na = na2; res = res2; }      // a second product of the same launch
            k_hi = (d.r + TILE - 1) / TILE * TILE;                  // (what lies behind, up to rp, is never written)
        }
    } else {
        // APPLY: neighbours differ in the rows of Q and share the piece of X
        const int sides = d.xo ? d.rp / TILE : (d.r + TILE - 1) / TILE;
        z = tile / n;
        const int t = tile - z * n, l = t / sides, o = t - l * sides;
        m0 = (MODE == APPLY_WIDE ? l : o) * TILE;
        n0 = (MODE == APPLY_WIDE ? o : l) * TILE;
        k_hi = (d.r + KSTEP - 1) / KSTEP * KSTEP;
    }
    int e = 0;
    float back = 1.f, up = 1.f;
    if constexpr (MODE != SYM) { norm_of(d, z, e, back); up = ldexpf(1.f, e); }
    const void *mp, *mlo = nullptr, *np, *nlo = nullptr;
    int mld, nld;
    const size_t esz = DT == 0 ? 4 : 2;
    if constexpr (DT == SRC_PAIR && MODE != SYM) { mp = np = d.xp + z * 2 * d.xplane; mlo = nlo = d.xp + z * 2 * d.xplane + d.xplane; mld = nld = d.xld; }
    constexpr bool MQ = MODE == SYM || MODE == APPLY_TALL, NQ = MODE == SYM || MODE == APPLY_WIDE;      // a symmetric matrix
    if constexpr (MQ) { mp = ma + (size_t)z * 2 * plane; mlo = ma + (size_t)z * 2 * plane + plane; mld = d.rp; }
    else if constexpr (DT != SRC_PAIR) { mp = (const char*)d.x + z * d.x_stride * esz; mld = d.cols; }
    if constexpr (NQ) { np = na + (size_t)z * 2 * plane; nlo = na + (size_t)z * 2 * plane + plane; nld = d.rp; }
    else if constexpr (DT != SRC_PAIR) { np = (const char*)d.x + z * d.x_stride * esz; nld = d.cols; }
    az_f4 acc[WT][WT];
    #pragma unroll
    for (int i = 0; i < WT; ++i)
        for (int j = 0; j < WT; ++j) acc[i][j] = az_f4{0.f, 0.f, 0.f, 0.f};
    // AHEAD steps of operands wait in registers: a step's products take a few hundred cycles, a load a few thousand
    constexpr int AHEAD = 2;
    OM om[AHEAD];
    ON on[AHEAD];
    #pragma unroll
    for (int u = 0; u < AHEAD; ++u)
        if (k_lo + u * KSTEP < k_hi) {
            om[u].load(mp, mlo, mld, m0, k_lo + u * KSTEP, d.rows, d.cols, tid);
            on[u].load(np, nlo, nld, n0, k_lo + u * KSTEP, d.rows, d.cols, tid);
        }
    const int mw = (wave & 1) * TILE / 2, nw = (wave >> 1) * TILE / 2;
    const auto step = [&](int k, OM& om, ON& on, int buf) __attribute__((always_inline)) {
        short* sm = lds + buf * STAGE;
        short* sn = sm + OM::PARTS * OM::HALVES;
        om.store(sm, m0, k, d.rows, d.cols, up, tid);
        on.store(sn, n0, k, d.rows, d.cols, up, tid);
        if (k + AHEAD * KSTEP < k_hi) {
            om.load(mp, mlo, mld, m0, k + AHEAD * KSTEP, d.rows, d.cols, tid);
            on.load(np, nlo, nld, n0, k + AHEAD * KSTEP, d.rows, d.cols, tid);
        }
        __syncthreads();                                             // (the other stage was last read before this barrier)
        #pragma unroll
        for (int kk = 0; kk < KSTEP; kk += 32) {
            az_i4 mf[WT][OM::PARTS];
            #pragma unroll
            for (int i = 0; i < WT; ++i)
                #pragma unroll
                for (int p = 0; p < OM::PARTS; ++p) mf[i][p] = OM::frag(sm, p, mw + i * 16, kk, lane);
            #pragma unroll
            for (int j = 0; j < WT; ++j) {
                az_i4 nf[ON::PARTS];
                #pragma unroll
                for (int p = 0; p < ON::PARTS; ++p) nf[p] = ON::frag(sn, p, nw + j * 16, kk, lane);
                #pragma unroll
                for (int i = 0; i < WT; ++i) {
                    acc[i][j] = az_mma<1>(mf[i][0], nf[0], acc[i][j]);
                    if constexpr (ON::PARTS == 2) acc[i][j] = az_mma<1>(mf[i][0], nf[1], acc[i][j]);
                    if constexpr (OM::PARTS == 2) acc[i][j] = az_mma<1>(mf[i][1], nf[0], acc[i][j]);
                }
            }
        }
    };
    #pragma unroll 1
    for (int k = k_lo; k < k_hi; k += AHEAD * KSTEP) {
        #pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            if (k + u * KSTEP < k_hi) step(k + u * KSTEP, om[u], on[u], u & 1);
    }
    #pragma unroll
    for (int i = 0; i < WT; ++i)
        #pragma unroll
        for (int j = 0; j < WT; ++j) {
            az_f4 v = acc[i][j];
            const int m = m0 + mw + i * 16 + q * 4, nn = n0 + nw + j * 16 + (lane & 15);
            if constexpr (MODE == SYM || GRAM) {
                if constexpr (GRAM) v *= back * back * (epi == EPI_PARTIAL ? 1.f : SA);
                else v *= 1.f / SA;                                  // (one factor is at scale SA: the result is at the other's)
                if (GRAM && epi == EPI_PARTIAL) { *(az_f4*)(d.partial + ((size_t)z * d.split + sp) * plane + (size_t)nn * d.rp + m) = v; continue; }
                if (MODE == SYM && epi == EPI_POLY) {                 // P = a I + b A + c A A at scale SA, and at SQ where it is Q
                    const az_s4 ah = *(const az_s4*)(ma + (size_t)z * 2 * plane + (size_t)nn * d.rp + m);
                    const az_s4 al = *(const az_s4*)(ma + (size_t)z * 2 * plane + plane + (size_t)nn * d.rp + m);
                    #pragma unroll
                    for (int t = 0; t < 4; ++t) v[t] = (m + t == nn ? d.a * SA : 0.f) + d.b * (az_from16<1>(ah[t]) + az_from16<1>(al[t])) + d.c * v[t];
                    if (res2) put_symmetric(d, res2, z, m, nn, m0 != n0, v * (SQ / SA));
                }
                if (res) put_symmetric(d, res, z, m, nn, m0 != n0, v);
            } else {
                // the result's line and position in memory: the positions m .. m + 3 of line nn
                if (d.xo) {                                          // (zero where the matrix is padded)
                    const float f = back * (1.f / SQ) * ldexpf(1.f, d.scale_exp);
                    short* hi = d.xo + z * 2 * d.xplane + (size_t)nn * d.xld + m;
                    az_s4 h, l;
                    #pragma unroll
                    for (int t = 0; t < 4; ++t) { short a, b; split(v[t] * f, a, b); h[t] = a; l[t] = b; }
                    *(az_s4*)hi = h;
                    *(az_s4*)(hi + d.xplane) = l;
                    continue;
                }
                const int nl = d.rows, np_ = d.cols;
                if (nn >= nl || m >= np_) continue;
                const float f = back * (1.f / SQ) * d.scale;
                const size_t at = (size_t)nn * d.cols + m;
                if (d.w) {
                    const float* w = d.w + z * d.w_stride + at;
                    float* o = (float*)d.out + z * d.out_stride + at;
                    if (m + 4 <= np_) { const az_f4 x = *(const az_f4_u*)w; *(az_f4_u*)o = x * d.keep + v * f; }
                    else for (int t = 0; t < 4; ++t) if (m + t < np_) o[t] = w[t] * d.keep + v[t] * f;
                } else if (d.out_dtype == AZ_F32) {
                    float* o = (float*)d.out + z * d.out_stride + at;
                    if (m + 4 <= np_) *(az_f4_u*)o = v * f;
                    else for (int t = 0; t < 4; ++t) if (m + t < np_) o[t] = v[t] * f;
                } else {
                    short* o = (short*)d.out + z * d.out_stride + at;
                    const bool h16 = d.out_dtype == AZ_F16;
                    az_s4 s;
                    for (int t = 0; t < 4; ++t) s[t] = h16 ? az_to16<1>(v[t] * f) : az_to16<2>(v[t] * f);
                    if (m + 4 <= np_) *(az_s4_u*)o = s;
                    else for (int t = 0; t < 4; ++t) if (m + t < np_) o[t] = s[t];
                }
            }
        }
}

// The slices of a contraction that was split, added in their order: A as pairs, both triangles.  Four entries of a row a
// thread, all slices' loads in flight.
__global__ void __launch_bounds__(256) az_ortho_join_kernel(OrthoDev d, int tile) {
    int ti, tj;
    lower_tile(blockIdx.x, ti, tj);
    const int z = blockIdx.z, i = (blockIdx.y * 256 + threadIdx.x) * 4;
    const size_t plane = (size_t)d.rp * d.rp;
    short* hi = d.A + (size_t)z * 2 * plane;
    short* lo = hi + plane;
    const int nn = ti * tile + i / tile, m = tj * tile + i % tile;
    const float* p = d.partial + (size_t)z * d.split * plane + (size_t)nn * d.rp + m;
    az_f4 v = {0.f, 0.f, 0.f, 0.f};
    #pragma unroll 8
    for (int s = 0; s < d.split; ++s) v += *(const az_f4*)(p + s * plane);
    az_s4 h, l;
    #pragma unroll
    for (int t = 0; t < 4; ++t) { short x, y; split(v[t] * SA, x, y); h[t] = x; l[t] = y; }
    *(az_s4*)(hi + (size_t)nn * d.rp + m) = h;
    *(az_s4*)(lo + (size_t)nn * d.rp + m) = l;
    if (ti != tj)
        #pragma unroll
        for (int t = 0; t < 4; ++t) { hi[(size_t)(m + t) * d.rp + nn] = h[t]; lo[(size_t)(m + t) * d.rp + nn] = l[t]; }
}

// no step at all: Q = I
__global__ void __launch_bounds__(256) az_ortho_identity_kernel(short* Q, int rp) {
    const size_t plane = (size_t)rp * rp;
    short* q = Q + (size_t)blockIdx.y * 2 * plane;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < 2 * plane; i += (size_t)gridDim.x * 256)
        q[i] = i < plane && i / rp == i % rp ? az_to16<1>(SQ) : (short)0;
}

// All of a stage's steps for matrices of up to R = 64 or 128 rows, one workgroup a matrix: A and P lie in LDS as pairs, Q in
// registers, A P takes A's place.  Launched one product at a time these cost a launch and a trip to L2 each (5 us) for
// 1 to 2 us of matrix instructions.  18 matrices of 128 rows: two steps 22 us, three 34.  One workgroup's chain of products:
// by counters its CU's matrix units work for a third of the time, its vector units for a third, LDS bank conflicts take 29 %
// (rows 16 halves longer instead of 8, a two-way conflict: a quarter more time), and barriers keep them apart.  A wave holds 16 columns of Q as operands: the product P Q leaves rows 4 g .. 4 g + 3 of
// the tiles 2 s, 2 s + 1 in lane group g, which is a fragment of step s whose contraction runs over those rows in that order,
// and P's rows are read in the same order.
template <int R> __global__ void __launch_bounds__(R * 4) az_ortho_iterate_kernel(OrthoDev d, int m) {
    constexpr int LD = R + 8, PLANE = R * LD, KS = R / 32, MT = R / 16, WM = R / 32, WN = 2, NTH = R * 4;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    short* const A = (short*)smem;                                   // [hi, lo][R][LD]
    short* const P = A + 2 * PLANE;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, q = lane >> 4, z = blockIdx.x;
    const size_t plane = (size_t)d.rp * d.rp;
    {
        const short* src = d.A + (size_t)z * 2 * plane;
        constexpr int PIECES = 2 * R * R / 8 / NTH;
        az_i4 v[PIECES];
        #pragma unroll
        for (int i = 0; i < PIECES; ++i) v[i] = ((const az_i4*)src)[tid + i * NTH];          // rp = R: both planes in one run
        #pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int e = (tid + i * NTH) * 8, part = e / (R * R), row = e % (R * R) / R;
            *(az_i4*)(A + part * PLANE + row * LD + e % R) = v[i];
        }
    }
    const int m0 = (wave & 1) * (R / 2), n0 = (wave >> 1) * 32;      // a wave's block of a product: R / 2 rows (M) by 32 (N)
    az_i4 qf[KS][2];                                                 // Q's columns 16 wave .. as operands
    az_f4 acc[WM][WN], qa[MT];
    const auto square = [&](const short* M, const short* N) __attribute__((always_inline)) {
        #pragma unroll
        for (int i = 0; i < WM; ++i)
            #pragma unroll
            for (int j = 0; j < WN; ++j) acc[i][j] = az_f4{0.f, 0.f, 0.f, 0.f};
        #pragma unroll
        for (int k = 0; k < R; k += 32) {
            az_i4 mf[WM][2], nf[WN][2];
            #pragma unroll
            for (int p = 0; p < 2; ++p) {
                #pragma unroll
                for (int i = 0; i < WM; ++i) mf[i][p] = az_row_frag<1>(M + p * PLANE, LD, m0 + i * 16, k, lane);
                #pragma unroll
                for (int j = 0; j < WN; ++j) nf[j][p] = az_row_frag<1>(N + p * PLANE, LD, n0 + j * 16, k, lane);
            }
            #pragma unroll
            for (int i = 0; i < WM; ++i)
                #pragma unroll
                for (int j = 0; j < WN; ++j) {
                    acc[i][j] = az_mma<1>(mf[i][0], nf[j][0], acc[i][j]);
                    acc[i][j] = az_mma<1>(mf[i][0], nf[j][1], acc[i][j]);
                    acc[i][j] = az_mma<1>(mf[i][1], nf[j][0], acc[i][j]);
                }
        }
    };
    // entry (n, m .. m + 3) of the symmetric result
    const auto put = [&](short* D, int i, int j, az_f4 v) __attribute__((always_inline)) {
        az_s4 h, l;
        #pragma unroll
        for (int t = 0; t < 4; ++t) { short x, y; split(v[t], x, y); h[t] = x; l[t] = y; }
        short* at = D + (n0 + j * 16 + (lane & 15)) * LD + m0 + i * 16 + q * 4;
        *(az_s4*)at = h;
        *(az_s4*)(at + PLANE) = l;
    };
    const auto put_all = [&](short* D, float scale) __attribute__((always_inline)) {
        #pragma unroll
        for (int i = 0; i < WM; ++i)
            #pragma unroll
            for (int j = 0; j < WN; ++j) put(D, i, j, acc[i][j] * scale);
    };
    #pragma unroll 1
    for (int step = 0; step < m; ++step) {
        __syncthreads();                                             // A is there
        square(A, A);
        #pragma unroll
        for (int i = 0; i < WM; ++i)
            #pragma unroll
            for (int j = 0; j < WN; ++j) {                           // P = a I + b A + c A A at scale SA
                const int nn = n0 + j * 16 + (lane & 15), mm = m0 + i * 16 + q * 4;
                const az_s4 h = *(const az_s4*)(A + nn * LD + mm), l = *(const az_s4*)(A + PLANE + nn * LD + mm);
                az_f4 v;
                #pragma unroll
                for (int t = 0; t < 4; ++t) v[t] = (mm + t == nn ? d.a * SA : 0.f) + d.b * (az_from16<1>(h[t]) + az_from16<1>(l[t])) + d.c * (acc[i][j][t] * (1.f / SA));
                put(P, i, j, v);
            }
        __syncthreads();
        // Q <- P Q (columns 16 wave ..); the first step's Q is P itself
        #pragma unroll
        for (int i = 0; i < MT; ++i) qa[i] = az_f4{0.f, 0.f, 0.f, 0.f};
        if (step == 0) {
            #pragma unroll
            for (int i = 0; i < MT; ++i) {
                const short* at = P + (wave * 16 + (lane & 15)) * LD + i * 16 + q * 4;
                const az_s4 h = *(const az_s4*)at, l = *(const az_s4*)(at + PLANE);
                #pragma unroll
                for (int t = 0; t < 4; ++t) qa[i][t] = (az_from16<1>(h[t]) + az_from16<1>(l[t])) * (SQ / SA);
            }
        } else {
            #pragma unroll
            for (int k = 0; k < KS; ++k)
                #pragma unroll
                for (int i = 0; i < MT; ++i) {
                    az_i4 pf[2];
                    #pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        const short* at = P + p * PLANE + (i * 16 + (lane & 15)) * LD + k * 32 + q * 4;
                        pf[p] = __builtin_bit_cast(az_i4, __builtin_shufflevector(*(const az_s4*)at, *(const az_s4*)(at + 16), 0, 1, 2, 3, 4, 5, 6, 7));
                    }
                    qa[i] = az_mma<1>(pf[0], qf[k][0], qa[i]);
                    qa[i] = az_mma<1>(pf[0], qf[k][1], qa[i]);
                    qa[i] = az_mma<1>(pf[1], qf[k][0], qa[i]);
                }
            #pragma unroll
            for (int i = 0; i < MT; ++i) qa[i] *= 1.f / SA;
        }
        #pragma unroll
        for (int k = 0; k < KS; ++k) {
            az_s8 h, l;
            #pragma unroll
            for (int t = 0; t < 8; ++t) { short x, y; split(qa[2 * k + (t >> 2)][t & 3], x, y); h[t] = x; l[t] = y; }
            qf[k][0] = __builtin_bit_cast(az_i4, h);
            qf[k][1] = __builtin_bit_cast(az_i4, l);
        }
        if (step + 1 < m) {
            square(A, P);                                            // A P
            __syncthreads();
            put_all(A, 1.f / SA);
            __syncthreads();
            square(A, P);                                            // A P P
            __syncthreads();
            put_all(A, 1.f / SA);
        }
    }
    short* out = d.Q + (size_t)z * 2 * plane + (size_t)(wave * 16 + (lane & 15)) * d.rp + q * 4;
    #pragma unroll
    for (int k = 0; k < KS; ++k)
        #pragma unroll
        for (int p = 0; p < 2; ++p) {
            const az_s8 v = __builtin_bit_cast(az_s8, qf[k][p]);
            *(az_s4*)(out + p * plane + k * 32) = __builtin_shufflevector(v, v, 0, 1, 2, 3);
            *(az_s4*)(out + p * plane + k * 32 + 16) = __builtin_shufflevector(v, v, 4, 5, 6, 7);
        }
}
template <int R> hipError_t iterate_in_lds(const OrthoDev& d, int n, int m, hipStream_t st) {
    constexpr size_t lds = (size_t)4 * R * (R + 8) * 2;
    if (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute((const void*)az_ortho_iterate_kernel<R>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    az_ortho_iterate_kernel<R><<<n, R * 4, lds, st>>>(d, m);
    return hipGetLastError();
}

// A whole call for matrices that fit one workgroup's LDS (up to 64 rows, 480 columns): momentum, norm, all steps, result.
// The long dimension is as cheap to multiply here as the short one, so the steps are the plain ones, X <- P X, on X as
// pairs; a wave owns its columns of X and replaces them in place.  Launched one product at a time the same call is 10 to 13
// launches of 4 to 5 us each: 64 x 225 fp32 63 us, here 32; 64 x 480 69 and 53 (one step: 24 and 24); 1000 x 64 x 480 547 and
// 234; 1000 x 27 x 128 231 and 78.  Bound by the chain of a step, 2 us and 2 more for 256 columns.
constexpr int SMALL_R = 64, SMALL_K = 480, SMALL_NT = 512;
struct SmallDev {
    const void* g;
    size_t g_stride;
    const float* mom;         // optimiser step: u = g + beta m' or m', m' = beta m + g
    float* mom_out;
    size_t m_stride, mo_stride;
    float beta;
    int nesterov, steps;
};
template <int DT, bool MOM> __global__ void __launch_bounds__(SMALL_NT, 2) az_ortho_small_kernel(OrthoDev d, SmallDev s) {
    constexpr int LD = SMALL_R + 8, PLANE = SMALL_R * LD;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    __shared__ double red[SMALL_NT / 64];
    short* const A = (short*)smem;                                   // [hi, lo][64][LD]
    short* const P = A + 2 * PLANE;
    short* const X = P + 2 * PLANE;                                  // [hi, lo][64][ldx], rows of k
    const int kp = (d.k + 31) / 32 * 32, ldx = kp + 8, xplane = SMALL_R * ldx;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, q = lane >> 4, z = blockIdx.x, count = d.rows * d.cols;
    const bool wide = d.rows <= d.cols;
    // The update is read twice, 32 elements a thread in flight: for its norm (and the momentum, which the second time is
    // read as written), and scaled into pairs.  Straight code that kept it in registers took longer: it runs once, at the
    // pace of instruction fetches.
    for (int i = tid; i < 2 * xplane / 8; i += SMALL_NT) ((az_i4*)X)[i] = az_i4{0, 0, 0, 0};
    constexpr int U = 8;                                             // quads
    const size_t go = z * s.g_stride, mo = z * s.m_stride, oo = z * s.mo_stride;
    const int quads = count / 4, left = count - quads * 4;
    const auto momentum = [&](float m, float v) __attribute__((always_inline)) { return s.beta * m + v; };
    const auto update = [&](float m, float v) __attribute__((always_inline)) { return s.nesterov ? v + s.beta * m : m; };
    double sum = 0.0;
    #pragma unroll 1
    for (int base = tid; base < quads; base += SMALL_NT * U) {
        az_f4 v[U], m[U];
        #pragma unroll
        for (int u = 0; u < U; ++u) {
            const size_t i = (size_t)min(base + u * SMALL_NT, quads - 1) * 4;
            v[u] = load4<DT>(s.g, go + i);
            if (MOM) m[u] = *(const az_f4_u*)(s.mom + mo + i);
        }
        #pragma unroll
        for (int u = 0; u < U; ++u)
            if (base + u * SMALL_NT < quads) {
                #pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (MOM) { m[u][e] = momentum(m[u][e], v[u][e]); v[u][e] = update(m[u][e], v[u][e]); }
                    sum += (double)v[u][e] * v[u][e];
                }
                if (MOM) *(az_f4_u*)(s.mom_out + oo + (size_t)(base + u * SMALL_NT) * 4) = m[u];
            }
    }
    float last = 0.f;                                                // the up to three elements behind the last quad
    if (tid < left) {
        const size_t i = (size_t)quads * 4 + tid;
        last = az_load<DT>(s.g, go + i);
        if (MOM) {
            const float m = momentum(s.mom[mo + i], last);
            s.mom_out[oo + i] = m;
            last = update(m, last);
        }
        sum += (double)last * last;
    }
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (lane == 0) red[wave] = sum;
    __syncthreads();
    sum = 0.0;
    for (int w = 0; w < SMALL_NT / 64; ++w) sum += red[w];
    const float up = ldexpf(1.f, d.scale_exp), down = ldexpf(1.f, -d.scale_exp);
    const double inv = (double)up / (sqrt(sum) + (double)d.eps);
    {
        const auto place = [&](int line, int pos, float v) __attribute__((always_inline)) {
            short* at = X + (wide ? line * ldx + pos : pos * ldx + line);
            split((float)(v * inv), at[0], at[xplane]);
        };
        int line = tid * 4 / d.cols, pos = tid * 4 - line * d.cols;
        const int dl = SMALL_NT * 4 / d.cols, dp = SMALL_NT * 4 - dl * d.cols;
        #pragma unroll 1
        for (int base = tid; base < quads; base += SMALL_NT * U) {
            az_f4 v[U], m[U];
            #pragma unroll
            for (int u = 0; u < U; ++u) {
                const size_t i = (size_t)min(base + u * SMALL_NT, quads - 1) * 4;
                v[u] = load4<DT>(s.g, go + i);
                if (MOM) m[u] = *(const az_f4_u*)(s.mom_out + oo + i);
            }
            #pragma unroll
            for (int u = 0; u < U; ++u) {
                if (base + u * SMALL_NT < quads) {                   // (the momentum of other elements is other threads')
                    int l = line, p = pos;
                    #pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        place(l, p, MOM ? update(m[u][e], v[u][e]) : v[u][e]);
                        if (++p == d.cols) { p = 0; ++l; }
                    }
                }
                line += dl; pos += dp;
                if (pos >= d.cols) { pos -= d.cols; ++line; }
            }
        }
        if (tid < left) { const int i = quads * 4 + tid, l = i / d.cols; place(l, i - l * d.cols, last); }
    }
    const int m0 = (wave & 3) * 16, n0 = (wave >> 2) * 32;           // a wave's 16 x 32 of A and P
    const auto pairs = [&](az_f4& acc, const az_i4* m, const az_i4* n) __attribute__((always_inline)) {
        acc = az_mma<1>(m[0], n[0], acc);
        acc = az_mma<1>(m[0], n[1], acc);
        acc = az_mma<1>(m[1], n[0], acc);
    };
    const auto rows_product = [&](az_f4* acc, const short* M, int ld, int plane, int len) __attribute__((always_inline)) {
        acc[0] = acc[1] = az_f4{0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < len; k += 32) {
            az_i4 mf[2], nf[2][2];
            #pragma unroll
            for (int p = 0; p < 2; ++p) {
                mf[p] = az_row_frag<1>(M + p * plane, ld, m0, k, lane);
                #pragma unroll
                for (int j = 0; j < 2; ++j) nf[j][p] = az_row_frag<1>(M + p * plane, ld, n0 + j * 16, k, lane);
            }
            #pragma unroll
            for (int j = 0; j < 2; ++j) pairs(acc[j], mf, nf[j]);
        }
    };
    const auto put = [&](short* at, int plane, az_f4 x) __attribute__((always_inline)) {
        az_s4 h, l;
        #pragma unroll
        for (int t = 0; t < 4; ++t) { short a, b; split(x[t], a, b); h[t] = a; l[t] = b; }
        *(az_s4*)at = h;
        *(az_s4*)(at + plane) = l;
    };
    #pragma unroll 1
    for (int step = 0; step < s.steps; ++step) {
        az_f4 acc[2], a[2];
        __syncthreads();                                             // X is there
        rows_product(a, X, ldx, xplane, kp);
        const float f = SA * down * down;
        #pragma unroll
        for (int j = 0; j < 2; ++j) { a[j] *= f; put(A + (n0 + j * 16 + (lane & 15)) * LD + m0 + q * 4, PLANE, a[j]); }
        __syncthreads();
        rows_product(acc, A, LD, PLANE, SMALL_R);
        #pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int nn = n0 + j * 16 + (lane & 15), mm = m0 + q * 4;
            #pragma unroll
            for (int t = 0; t < 4; ++t) acc[j][t] = (mm + t == nn ? d.a * SA : 0.f) + d.b * a[j][t] + d.c * (acc[j][t] * (1.f / SA));
            put(P + nn * LD + mm, PLANE, acc[j]);
        }
        __syncthreads();
        // X <- P X, 16 columns at a time; the last step's go to the result
        az_i4 pf[4][2][2];
        #pragma unroll
        for (int j = 0; j < 4; ++j)
            #pragma unroll
            for (int k = 0; k < 2; ++k)
                #pragma unroll
                for (int p = 0; p < 2; ++p) pf[j][k][p] = az_row_frag<1>(P + p * PLANE, LD, j * 16, k * 32, lane);
        #pragma unroll 1
        for (int c = wave * 16; c < kp; c += SMALL_NT / 64 * 16) {
            az_f4 x[4];
            #pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = az_f4{0.f, 0.f, 0.f, 0.f};
            #pragma unroll
            for (int k = 0; k < 2; ++k) {
                az_i4 xf[2];
                #pragma unroll
                for (int p = 0; p < 2; ++p) xf[p] = az_col_frag<1>(X + p * xplane, ldx, k * 32, c, lane);
                #pragma unroll
                for (int j = 0; j < 4; ++j) pairs(x[j], xf, pf[j][k]);
            }
            #pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int row = j * 16 + (lane & 15), col = c + q * 4;
                if (step + 1 < s.steps) { put(X + row * ldx + col, xplane, x[j] * (1.f / SA)); continue; }
                if (row >= d.r) continue;
                const az_f4 y = x[j] * (down * (1.f / SA) * d.scale);
                if (wide && col + 4 <= d.k) {
                    const size_t at = (size_t)row * d.cols + col;
                    if (MOM) *(az_f4_u*)((float*)d.out + z * d.out_stride + at) = *(const az_f4_u*)(d.w + z * d.w_stride + at) * d.keep + y;
                    else if constexpr (DT == 0) *(az_f4_u*)((float*)d.out + z * d.out_stride + at) = y;
                    else *(az_s4_u*)((short*)d.out + z * d.out_stride + at) = az_s4{az_to16<DT>(y[0]), az_to16<DT>(y[1]), az_to16<DT>(y[2]), az_to16<DT>(y[3])};
                    continue;
                }
                #pragma unroll
                for (int t = 0; t < 4; ++t) {
                    if (col + t >= d.k) continue;
                    const size_t at = wide ? (size_t)row * d.cols + col + t : (size_t)(col + t) * d.cols + row;
                    if (MOM) ((float*)d.out)[z * d.out_stride + at] = d.w[z * d.w_stride + at] * d.keep + y[t];
                    else az_store<DT>(d.out, z * d.out_stride + at, y[t]);
                }
            }
        }
    }
}
bool fits_small(int r, int k, int steps) { return r <= SMALL_R && k <= SMALL_K && steps > 0; }
template <int DT, bool MOM> hipError_t small(OrthoDev d, const SmallDev& s, int n, hipStream_t st) {
    d.scale_exp = std::ilogb(std::sqrt((double)d.k)) + 2;            // an iterate's elements: about 1 / sqrt(k)
    const size_t lds = (size_t)2 * SMALL_R * ((d.k + 31) / 32 * 32 + 8) * 2 + (size_t)4 * SMALL_R * (SMALL_R + 8) * 2;
    if (lds > 60 * 1024) {
        const hipError_t e = hipFuncSetAttribute((const void*)az_ortho_small_kernel<DT, MOM>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    az_ortho_small_kernel<DT, MOM><<<n, SMALL_NT, lds, st>>>(d, s);
    return hipGetLastError();
}

struct Plan {
    int n, rows, cols, r, k, rp, kp, apply_tile, low, slices, split, stage;
    bool muon, restart, small;
    size_t off_sq, off_u, off_x1, off_mat, off_partial, bytes;
    size_t pair_bytes, iter_bytes;
};

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// Largest |a + b y + c y^2| that the steps meet from singular values of up to 1 on, y their squares; negative where a value passes
// MOST_ON_THE_WAY ahead of a step, or a factor MOST_FACTOR.  A step maps 0 .. x onto 0 .. the largest |t (a + b t^2 + c t^4)| for
// t <= x, which lies at x or where the derivative is 0.  In that range, at the pairs' scales and in fp16 (65504): A <= 49 SA,
// P <= 200 SA, P A (formed where another step follows) <= 49 SA, an iterate's elements <= 7 * 2^13; Q, a product of P's: make_plan.
constexpr double MOST_ON_THE_WAY = 7.0, MOST_FACTOR = 200.0;
double largest_factor(double a, double b, double c, int steps) {
    const auto factor = [&](double y) { return std::fabs(a + y * (b + y * c)); };
    double most = 1.0, largest = 0.0;
    for (int i = 0; i < steps; ++i) {
        if (most > MOST_ON_THE_WAY) return -1.0;
        const double end = most * most, disc = 9.0 * b * b - 20.0 * a * c;
        double at[3] = {end, 0.0, 0.0}, peak = 0.0;                  // derivatives: a + 3 b y + 5 c y^2, and b + 2 c y
        if (c != 0.0) {
            peak = -b / (2.0 * c);
            if (disc >= 0.0) { at[1] = (-3.0 * b + std::sqrt(disc)) / (10.0 * c); at[2] = (-3.0 * b - std::sqrt(disc)) / (10.0 * c); }
        } else if (b != 0.0) at[1] = -a / (3.0 * b);
        most = 0.0;
        for (const double y : at) if (y > 0.0 && y <= end) most = std::fmax(most, std::sqrt(y) * factor(y));
        largest = std::fmax(largest, std::fmax(std::fabs(a), std::fmax(factor(end), peak > 0.0 && peak <= end ? factor(peak) : 0.0)));
    }
    return largest > MOST_FACTOR ? -1.0 : largest;
}

// Slices of the contraction of X X^T.  In steps of 64 (1.4 us where a workgroup has its CU to itself; two take 1.7 times as
// long): what the fullest CU does, two more to begin a workgroup, five for the launch that joins the slices, and the slices'
// traffic (16 KB a tile written and read).  2 x 4096 x 1024 (272 tiles on 256 CUs, 64 steps): a slice 696 us a call, two 677,
// four 653; 40 x 256 x 2304 (400 tiles, 36 steps): one 587, two 613; 18 x 128 x 1152 (54 tiles, 18 steps): one 115, four 107.
int split_of(long long tiles, int steps) {
    int best = 1;
    double cost = 0.0;
    for (int s = 1; s <= 64 && s <= steps; s *= 2) {
        const long long w = (tiles * s + 255) / 256;
        const double t = ((double)(w / 2) * 1.7 + (double)(w % 2)) * ((steps + s - 1) / s + 2) + (s > 1 ? 5.0 + (double)tiles * s * 0.0047 : 0.0);
        if (s == 1 || t < cost) { cost = t; best = s; }
    }
    return best;
}

Plan make_plan(int n, int rows, int cols, int dtype, int steps, float a, float b, float c, bool muon) {
    Plan p = {};
    p.n = n; p.rows = rows; p.cols = cols; p.muon = muon;
    p.r = rows < cols ? rows : cols;
    p.k = rows < cols ? cols : rows;
    const int t = (p.r + 63) / 64;
    p.low = t * (t + 1) / 2;
    p.rp = p.r <= 64 ? 64 : (p.r + 127) / 128 * 128;
    p.kp = (p.k + 127) / 128 * 128;
    // Q X in tiles of 128 where they fill the chip (figures at az_ortho_product_kernel)
    p.apply_tile = p.rp % 128 == 0 && (long long)((p.k + 127) / 128) * ((p.r + 127) / 128) * n >= 256 ? 128 : 64;
    const long long count = (long long)rows * cols;
    p.slices = (int)(count / 4096 < 1 ? 1 : count / 4096 > MAX_SLICES ? MAX_SLICES : count / 4096);
    while (p.slices > 64 && (long long)p.slices * n > 2048) p.slices /= 2;
    p.split = split_of((long long)p.low * n, (p.k + 63) / 64);
    // Steps between two formations of X.  fp32 results and the optimiser step's weights: two (comment at the top; 40 x 256 x 2304
    // with three 493 us a step, with two 579).  16-bit results: three, off by at most 8e-5 where half a step of fp16 is 2e-4 and of bf16
    // 1.7e-3 (relative norms over 128 x 1152 .. 600 x 200, one to eight strong directions a thousand to ten thousand times the
    // rest, where fp32 products are off by as much); all five at once leave 1e-3 to 7e-3 there.  18 x 128 x 1152 bf16: five
    // 86 us a call, three 106, two 131; 300 x 128 x 1152: five 227, three 390.  Fewer where the coefficients would take Q out of fp16's range.
    p.stage = dtype == AZ_F32 ? 2 : 3;
    const double f = largest_factor(a, b, c, steps);
    while (p.stage > 1 && std::pow(f, p.stage) * SQ > 30000.0) --p.stage;
    p.restart = steps > p.stage;
    p.pair_bytes = up256((size_t)n * 2 * p.rp * p.rp * 2);
    if ((p.small = fits_small(p.r, p.k, steps))) return p;           // (no workspace)
    size_t o = 0;
    p.off_sq = o; o += up256((size_t)n * p.slices * 8);
    p.off_u = o; if (muon) o += up256((size_t)n * count * 4);
    // iterates: of three stages and more the middle ones read one and write the other
    p.off_x1 = o; if (p.restart) o += (steps > 2 * p.stage ? 2 : 1) * (p.iter_bytes = up256((size_t)n * 2 * p.rp * p.kp * 2));
    p.off_mat = o; o += 5 * p.pair_bytes;
    p.off_partial = o; if (p.split > 1) o += up256((size_t)n * p.split * p.rp * p.rp * 4);
    p.bytes = o;
    return p;
}

struct Pairs { const short *m, *n; short* out; };                    // one product: operands, result
// grid x: tiles of a matrix, z: matrices (one dimension of the launch), y: slices or products
template <int TILE, int DT, int MODE> hipError_t product(const OrthoDev& d, dim3 grid, Pairs one, Pairs two, int epi, hipStream_t st) {
    constexpr int MS = MODE == SYM || MODE == APPLY_TALL ? SRC_PAIR : DT, NS = MODE == SYM || MODE == APPLY_WIDE ? SRC_PAIR : DT;
    typedef Operand<TILE, MS, !(MODE == GRAM_TALL || MODE == APPLY_WIDE)> OM;
    typedef Operand<TILE, NS, MODE != GRAM_TALL> ON;
    const size_t lds = 2 * 2 * ((size_t)OM::PARTS * OM::HALVES + (size_t)ON::PARTS * ON::HALVES);
    if (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute((const void*)az_ortho_product_kernel<TILE, DT, MODE>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    az_ortho_product_kernel<TILE, DT, MODE><<<dim3(grid.x * grid.z, grid.y), 256, lds, st>>>(d, one.m, one.n, one.out, two.m, two.n, two.out, epi, (int)grid.x);
    return hipGetLastError();
}

template <int TILE, int DT> hipError_t gram(const Plan& p, const OrthoDev& d, hipStream_t st) {
    const dim3 grid(p.low, p.split, p.n);
    const int epi = p.split > 1 ? EPI_PARTIAL : EPI_PAIR;
    const Pairs x = {nullptr, nullptr, d.A};
    hipError_t e = p.rows <= p.cols ? product<TILE, DT, GRAM_WIDE>(d, grid, x, Pairs{}, epi, st) : product<TILE, DT, GRAM_TALL>(d, grid, x, Pairs{}, epi, st);
    if (e == hipSuccess && p.split > 1) {
        az_ortho_join_kernel<<<dim3(p.low, TILE * TILE / 1024, p.n), 256, 0, st>>>(d, TILE);
        e = hipGetLastError();
    }
    return e;
}
template <int TILE, int DT> hipError_t apply(const Plan& p, const OrthoDev& d, hipStream_t st) {
    const dim3 grid(d.xo ? p.kp / TILE * (p.rp / TILE) : (p.k + TILE - 1) / TILE * ((p.r + TILE - 1) / TILE), 1, p.n);
    return p.rows <= p.cols ? product<TILE, DT, APPLY_WIDE>(d, grid, Pairs{nullptr, d.Q, nullptr}, Pairs{}, 0, st)
                            : product<TILE, DT, APPLY_TALL>(d, grid, Pairs{d.Q, nullptr, nullptr}, Pairs{}, 0, st);
}
hipError_t gram_dt(int dt, const Plan& p, const OrthoDev& d, hipStream_t st) {
    return dt == SRC_PAIR ? gram<64, SRC_PAIR>(p, d, st) : dt == AZ_F32 ? gram<64, 0>(p, d, st) : dt == AZ_F16 ? gram<64, 1>(p, d, st) : gram<64, 2>(p, d, st);
}
template <int TILE> hipError_t apply_dt(int dt, const Plan& p, const OrthoDev& d, hipStream_t st) {
    return dt == SRC_PAIR ? apply<TILE, SRC_PAIR>(p, d, st) : dt == AZ_F32 ? apply<TILE, 0>(p, d, st) : dt == AZ_F16 ? apply<TILE, 1>(p, d, st) : apply<TILE, 2>(p, d, st);
}

// `m` steps on A: leaves Q
hipError_t iterate(const Plan& p, OrthoDev& d, int m, hipStream_t st) {
    const dim3 one(p.low, 1, p.n), two(p.low, 2, p.n);
    hipError_t e = hipSuccess;
#define RUN(call) do { if (e == hipSuccess) e = (call); } while (0)
    if (m == 0) { az_ortho_identity_kernel<<<dim3(64, p.n), 256, 0, st>>>(d.Q, p.rp); return hipGetLastError(); }
    if (p.rp == 64) return iterate_in_lds<64>(d, p.n, m, st);
    if (p.rp == 128) return iterate_in_lds<128>(d, p.n, m, st);
    for (int i = 0; i < m; ++i) {
        const bool first = i == 0, last = i + 1 == m;
        // P; the first step's is Q too
        RUN((product<64, 0, SYM>(d, one, Pairs{d.A, d.A, first && last ? nullptr : d.P}, Pairs{nullptr, nullptr, first ? d.Q : nullptr}, EPI_POLY, st)));
        const Pairs q = {d.Q, d.P, d.Q2};
        if (!last) {
            RUN((product<64, 0, SYM>(d, first ? one : two, Pairs{d.A, d.P, d.T}, first ? Pairs{} : q, EPI_PAIR, st)));
            RUN((product<64, 0, SYM>(d, one, Pairs{d.T, d.P, d.A}, Pairs{}, EPI_PAIR, st)));
        } else if (!first) RUN((product<64, 0, SYM>(d, one, q, Pairs{}, EPI_PAIR, st)));
        if (!first) { short* t = d.Q; d.Q = d.Q2; d.Q2 = t; }
    }
#undef RUN
    return e;
}

hipError_t run_plan(const Plan& p, OrthoDev d, int dtype, int steps, unsigned char* ws, hipStream_t st) {
    short* const x[2] = {(short*)(ws + p.off_x1), (short*)(ws + p.off_x1 + p.iter_bytes)};
    const bool wide = p.rows <= p.cols;
    d.xld = wide ? p.kp : p.rp;
    d.xplane = (size_t)p.rp * p.kp;
    const int se = std::ilogb(std::sqrt((double)p.k)) + 2;           // an iterate's elements: about 1 / sqrt(k)
    d.scale_exp = se < 13 ? se : 13;
    hipError_t e = hipSuccess;
    int done = 0, which = 0;
    do {
        // stages of p.stage steps, a shorter one last: A's error is relative to its largest eigenvalue, which the first
        // stage starts far below 1 (|X0|_F = 1 spread over the singular values) and the later ones near 1
        const int left = steps - done, m = left < p.stage ? left : p.stage;
        done += m;
        if (m > 0) e = gram_dt(dtype, p, d, st);
        if (e == hipSuccess) e = iterate(p, d, m, st);
        d.xo = done < steps ? x[which] : nullptr;
        if (e == hipSuccess) e = p.apply_tile == 64 ? apply_dt<64>(dtype, p, d, st) : apply_dt<128>(dtype, p, d, st);
        d.xp = x[which]; dtype = SRC_PAIR; d.sq = nullptr;
        which ^= 1;
    } while (e == hipSuccess && done < steps);
    return e;
}

int check_common(int n, int rows, int cols, int steps, float a, float b, float c, float eps) {
    if (n < 0) return ofail(AZ_E_ARG, "%d matrices", n);
    if (n > 65535) return ofail(AZ_E_ARG, "%d matrices are too many for one call (65535)", n);
    if (rows < 1 || cols < 1) return ofail(AZ_E_ARG, "matrix %d x %d", rows, cols);
    if ((long long)rows * cols > 0x7fffffffll) return ofail(AZ_E_ARG, "matrix %d x %d has too many elements", rows, cols);
    if ((rows < cols ? cols : rows) > 1 << 24) return ofail(AZ_E_ARG, "the longer side of %d x %d is beyond 2^24", rows, cols);
    if ((rows < cols ? rows : cols) > 8192) return ofail(AZ_E_ARG, "the shorter side of %d x %d is beyond 8192", rows, cols);
    if (steps < 0 || steps > 100) return ofail(AZ_E_ARG, "%d steps (0..100)", steps);
    if (!(std::fabs(a) + std::fabs(b) + std::fabs(c) <= 32.f)) return ofail(AZ_E_ARG, "coefficients %g, %g, %g: their magnitudes sum beyond 32", a, b, c);
    if (largest_factor(a, b, c, steps) < 0.0) return ofail(AZ_E_ARG, "coefficients %g, %g, %g: %d steps take singular values beyond %g or enlarge one more than %g times", a, b, c, steps, MOST_ON_THE_WAY, MOST_FACTOR);
    if (!(eps >= 0.f) || std::isinf(eps)) return ofail(AZ_E_ARG, "eps %g", eps);
    return AZ_OK;
}
// a launch takes fewer than 2^32 threads
int check_tiles(const Plan& p) {
    const long long tiles = (long long)(p.kp / p.apply_tile) * (p.rp / p.apply_tile);
    if (!p.small && (tiles > p.low ? tiles : p.low) * p.n >= 1 << 24) return ofail(AZ_E_ARG, "%d matrices of %d x %d are too many tiles for one call", p.n, p.rows, p.cols);
    return AZ_OK;
}
int check_ortho(const az_orthogonalize_args* p) {
    if (!p) return ofail(AZ_E_ARG, "null argument: args");
    const int rc = check_common(p->n, p->rows, p->cols, p->steps, p->a, p->b, p->c, p->eps);
    if (rc != AZ_OK) return rc;
    if (p->dtype != AZ_F32 && p->dtype != AZ_F16 && p->dtype != AZ_BF16) return ofail(AZ_E_ARG, "element type %d unknown (AZ_F32, AZ_F16, AZ_BF16)", p->dtype);
    return AZ_OK;
}
int check_muon(const az_muon_step_args* p) {
    if (!p) return ofail(AZ_E_ARG, "null argument: args");
    const int rc = check_common(p->n, p->rows, p->cols, p->steps, p->a, p->b, p->c, p->eps);
    if (rc != AZ_OK) return rc;
    if (p->grad_dtype != AZ_F32 && p->grad_dtype != AZ_F16 && p->grad_dtype != AZ_BF16) return ofail(AZ_E_ARG, "element type %d unknown (AZ_F32, AZ_F16, AZ_BF16)", p->grad_dtype);
    return AZ_OK;
}
// matrices that are written may not overlap each other: strides of at least a matrix
int check_stride(const char* name, int64_t stride, int n, int rows, int cols) {
    if (n > 1 && stride < (int64_t)rows * cols) return ofail(AZ_E_ARG, "%s: stride %lld is shorter than a %d x %d matrix", name, (long long)stride, rows, cols);
    return AZ_OK;
}
// the bytes a batch of matrices spans
struct Span { const char *lo, *hi; int64_t stride; };
Span span_of(const void* p, int64_t stride, int n, int rows, int cols, int esz) {
    const char* c = (const char*)p;
    return {c, c + ((int64_t)(n - 1) * stride + (int64_t)rows * cols) * esz, stride};
}
bool meet(const Span& a, const Span& b) { return a.lo < b.hi && b.lo < a.hi; }
bool same(const Span& a, const Span& b) { return a.lo == b.lo && a.stride == b.stride; }
int check_ws(const void* ws, size_t have, size_t need) {
    if (!ws) return ofail(AZ_E_ARG, "null argument: workspace");
    if ((size_t)ws % 256) return ofail(AZ_E_ARG, "workspace needs 256-byte alignment");
    if (have < need) return ofail(AZ_E_CAPACITY, "workspace has %zu bytes, the call needs %zu", have, need);
    return AZ_OK;
}

int run(const Plan& p, OrthoDev d, int dtype, int steps, unsigned char* ws, hipStream_t st, const char* who) {
    d.rows = p.rows; d.cols = p.cols; d.r = p.r; d.k = p.k; d.rp = p.rp; d.slices = p.slices; d.split = p.split;
    d.sq = (const double*)(ws + p.off_sq);
    short** m[5] = {&d.A, &d.P, &d.T, &d.Q, &d.Q2};
    for (int i = 0; i < 5; ++i) *m[i] = (short*)(ws + p.off_mat + i * p.pair_bytes);
    d.partial = (float*)(ws + p.off_partial);
    const hipError_t e = run_plan(p, d, dtype, steps, ws, st);
    if (e != hipSuccess) return ofail(AZ_E_HIP, "%s: launch failed: %s", who, hipGetErrorString(e));
    return AZ_OK;
}

}  // namespace

extern "C" size_t az_orthogonalize_workspace(const az_orthogonalize_args* p) {
    if (check_ortho(p) != AZ_OK) return 0;
    const Plan plan = make_plan(p->n, p->rows, p->cols, p->dtype, p->steps, p->a, p->b, p->c, false);
    return check_tiles(plan) == AZ_OK ? plan.bytes + 256 : 0;
}
extern "C" size_t az_muon_step_workspace(const az_muon_step_args* p) {
    if (check_muon(p) != AZ_OK) return 0;
    const Plan plan = make_plan(p->n, p->rows, p->cols, AZ_F32, p->steps, p->a, p->b, p->c, true);
    return check_tiles(plan) == AZ_OK ? plan.bytes + 256 : 0;
}

extern "C" int az_orthogonalize_dev(const az_orthogonalize_args* p, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_ortho(p);
    if (rc != AZ_OK) return rc;
    if (p->n == 0) return AZ_OK;
    if (!p->update) return ofail(AZ_E_ARG, "null argument: update");
    if (!p->out) return ofail(AZ_E_ARG, "null argument: out");
    if (((size_t)p->update | (size_t)p->out) % (p->dtype == AZ_F32 ? 4 : 2)) return ofail(AZ_E_ARG, "a tensor is not aligned to its element type");
    if ((rc = check_stride("update", p->update_stride, p->n, p->rows, p->cols)) != AZ_OK || (rc = check_stride("out", p->out_stride, p->n, p->rows, p->cols)) != AZ_OK) return rc;
    const int esz = p->dtype == AZ_F32 ? 4 : 2;
    // (a tile of the result is written while other workgroups still read the update)
    if (meet(span_of(p->update, p->update_stride, p->n, p->rows, p->cols, esz), span_of(p->out, p->out_stride, p->n, p->rows, p->cols, esz)))
        return ofail(AZ_E_ARG, "out overlaps update");
    const Plan plan = make_plan(p->n, p->rows, p->cols, p->dtype, p->steps, p->a, p->b, p->c, false);
    if ((rc = check_tiles(plan)) != AZ_OK || (rc = check_ws(workspace, workspace_bytes, plan.bytes + 256)) != AZ_OK) return rc;
    AzDeviceGuard dev(p->device);
    if (!dev.ok) return ofail(AZ_E_HIP, "device %d cannot be used (no HIP device: libazhip has no CPU fallback)", p->device);
    (void)hipGetLastError();                                         // (an earlier call's error is not this one's)
    unsigned char* ws = (unsigned char*)workspace;
    hipStream_t st = (hipStream_t)stream;
    OrthoDev d = {};
    d.x = p->update; d.x_stride = p->update_stride;
    d.eps = p->eps; d.a = p->a; d.b = p->b; d.c = p->c;
    d.out = p->out; d.out_stride = p->out_stride; d.out_dtype = p->dtype; d.scale = p->scale;
    if (plan.small) {
        const SmallDev s = {p->update, (size_t)p->update_stride, nullptr, nullptr, 0, 0, 0.f, 0, p->steps};
        d.rows = plan.rows; d.cols = plan.cols; d.r = plan.r; d.k = plan.k;
        const hipError_t e = p->dtype == AZ_F32 ? small<0, false>(d, s, p->n, st) : p->dtype == AZ_F16 ? small<1, false>(d, s, p->n, st) : small<2, false>(d, s, p->n, st);
        return e == hipSuccess ? AZ_OK : ofail(AZ_E_HIP, "az_orthogonalize_dev: launch failed: %s", hipGetErrorString(e));
    }
    double* sq = (double*)(ws + plan.off_sq);
    const dim3 grid(plan.slices, p->n);
    const int count = p->rows * p->cols;
    if (p->dtype == AZ_F32) az_ortho_norm_kernel<0, false><<<grid, 256, 0, st>>>(p->update, p->update_stride, count, plan.slices, sq, nullptr, 0, nullptr, 0, nullptr, 0.f, 0);
    else if (p->dtype == AZ_F16) az_ortho_norm_kernel<1, false><<<grid, 256, 0, st>>>(p->update, p->update_stride, count, plan.slices, sq, nullptr, 0, nullptr, 0, nullptr, 0.f, 0);
    else az_ortho_norm_kernel<2, false><<<grid, 256, 0, st>>>(p->update, p->update_stride, count, plan.slices, sq, nullptr, 0, nullptr, 0, nullptr, 0.f, 0);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return ofail(AZ_E_HIP, "az_orthogonalize_dev: launch failed: %s", hipGetErrorString(e));
    return run(plan, d, p->dtype, p->steps, ws, st, "az_orthogonalize_dev");
}

extern "C" int az_muon_step_dev(const az_muon_step_args* p, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_muon(p);
    if (rc != AZ_OK) return rc;
    if (p->n == 0) return AZ_OK;
    if (!p->grad) return ofail(AZ_E_ARG, "null argument: grad");
    if (!p->weight) return ofail(AZ_E_ARG, "null argument: weight");
    if (!p->momentum) return ofail(AZ_E_ARG, "null argument: momentum");
    if (!p->weight_out) return ofail(AZ_E_ARG, "null argument: weight_out");
    if (!p->momentum_out) return ofail(AZ_E_ARG, "null argument: momentum_out");
    if ((size_t)p->grad % (p->grad_dtype == AZ_F32 ? 4 : 2) || ((size_t)p->weight | (size_t)p->momentum | (size_t)p->weight_out | (size_t)p->momentum_out) % 4)
        return ofail(AZ_E_ARG, "a tensor is not aligned to its element type");
    const struct { const char* name; int64_t s; } strides[5] = {{"grad", p->grad_stride}, {"weight", p->weight_stride}, {"momentum", p->momentum_stride},
                                                                 {"weight_out", p->weight_out_stride}, {"momentum_out", p->momentum_out_stride}};
    for (const auto& s : strides) if ((rc = check_stride(s.name, s.s, p->n, p->rows, p->cols)) != AZ_OK) return rc;
    const Span g = span_of(p->grad, p->grad_stride, p->n, p->rows, p->cols, p->grad_dtype == AZ_F32 ? 4 : 2);
    const Span w = span_of(p->weight, p->weight_stride, p->n, p->rows, p->cols, 4), m = span_of(p->momentum, p->momentum_stride, p->n, p->rows, p->cols, 4);
    const Span wo = span_of(p->weight_out, p->weight_out_stride, p->n, p->rows, p->cols, 4), mo = span_of(p->momentum_out, p->momentum_out_stride, p->n, p->rows, p->cols, 4);
    if ((meet(w, wo) && !same(w, wo)) || (meet(m, mo) && !same(m, mo)) || meet(wo, mo) || meet(wo, m) || meet(mo, w) || meet(g, wo) || meet(g, mo))
        return ofail(AZ_E_ARG, "an output overlaps another tensor (in place means the same address and stride)");
    const Plan plan = make_plan(p->n, p->rows, p->cols, AZ_F32, p->steps, p->a, p->b, p->c, true);
    if ((rc = check_tiles(plan)) != AZ_OK || (rc = check_ws(workspace, workspace_bytes, plan.bytes + 256)) != AZ_OK) return rc;
    AzDeviceGuard dev(p->device);
    if (!dev.ok) return ofail(AZ_E_HIP, "device %d cannot be used (no HIP device: libazhip has no CPU fallback)", p->device);
    (void)hipGetLastError();                                         // (an earlier call's error is not this one's)
    unsigned char* ws = (unsigned char*)workspace;
    hipStream_t st = (hipStream_t)stream;
    OrthoDev d = {};
    d.eps = p->eps; d.a = p->a; d.b = p->b; d.c = p->c;
    d.out = p->weight_out; d.out_stride = p->weight_out_stride; d.out_dtype = AZ_F32; d.scale = -p->lr * p->scale;
    d.w = p->weight; d.w_stride = p->weight_stride; d.keep = 1.f - p->lr * p->weight_decay;
    if (plan.small) {
        const SmallDev s = {p->grad, (size_t)p->grad_stride, p->momentum, p->momentum_out, (size_t)p->momentum_stride, (size_t)p->momentum_out_stride, p->beta, p->nesterov, p->steps};
        d.rows = plan.rows; d.cols = plan.cols; d.r = plan.r; d.k = plan.k;
        const hipError_t e = p->grad_dtype == AZ_F32 ? small<0, true>(d, s, p->n, st) : p->grad_dtype == AZ_F16 ? small<1, true>(d, s, p->n, st) : small<2, true>(d, s, p->n, st);
        return e == hipSuccess ? AZ_OK : ofail(AZ_E_HIP, "az_muon_step_dev: launch failed: %s", hipGetErrorString(e));
    }
    double* sq = (double*)(ws + plan.off_sq);
    float* u = (float*)(ws + plan.off_u);
    const dim3 grid(plan.slices, p->n);
    const int count = p->rows * p->cols;
#define NORM(DT) az_ortho_norm_kernel<DT, true><<<grid, 256, 0, st>>>(p->grad, p->grad_stride, count, plan.slices, sq, p->momentum, p->momentum_stride, \
                                                                p->momentum_out, p->momentum_out_stride, u, p->beta, p->nesterov)
    if (p->grad_dtype == AZ_F32) NORM(0);
    else if (p->grad_dtype == AZ_F16) NORM(1);
    else NORM(2);
#undef NORM
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return ofail(AZ_E_HIP, "az_muon_step_dev: launch failed: %s", hipGetErrorString(e));
    d.x = u; d.x_stride = count;
    return run(plan, d, AZ_F32, p->steps, ws, st, "az_muon_step_dev");
}
