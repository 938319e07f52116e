// Shared by the learner's operators (policy_loss.hip, orthogonalize.hip): element types, the matrix-instruction
// fragments both are written in, and the host-side error hooks.
//
// A fragment is 16 bytes a lane: 8 elements of a 16-bit type or 4 of fp32.  One step of a product runs over KS = 4 * EP
// elements of the contraction (32 or 16): lane l holds elements EP * (l / 16) .. + EP - 1 of row l % 16 (operand A) or
// of column l % 16 (operand B).  For fp32 that is four v_mfma_f32_16x16x4_f32 whose k = l / 16 stands for element
// EP * (l / 16) + j in the j-th of them: any order of the contraction is right as long as both operands share it.
// The result of a 16 x 16 tile: lane l holds rows 4 * (l / 16) .. + 3 of column l % 16.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

typedef float az_f4 __attribute__((ext_vector_type(4)));
typedef _Float16 az_h8 __attribute__((ext_vector_type(8)));
typedef __bf16 az_b8 __attribute__((ext_vector_type(8)));
typedef short az_s4 __attribute__((ext_vector_type(4)));
typedef short az_s8 __attribute__((ext_vector_type(8)));
typedef int az_i4 __attribute__((ext_vector_type(4)));
// the same 16 bytes where only the element's own alignment is known (the hardware takes such loads and stores)
typedef float az_f4_u __attribute__((ext_vector_type(4), aligned(4)));
typedef short az_s8_u __attribute__((ext_vector_type(8), aligned(2)));
typedef short az_s4_u __attribute__((ext_vector_type(4), aligned(2)));

template <int DT> struct AzElem;                                     // DT: AZ_F32 / AZ_F16 / AZ_BF16
template <> struct AzElem<0> { typedef float T; static constexpr int EP = 4, KS = 16; };
template <> struct AzElem<1> { typedef _Float16 T; static constexpr int EP = 8, KS = 32; };
template <> struct AzElem<2> { typedef __bf16 T; static constexpr int EP = 8, KS = 32; };

template <int DT> __device__ __forceinline__ az_f4 az_mma(az_i4 a, az_i4 b, az_f4 c) {
    if constexpr (DT == 0) {
        const az_f4 x = __builtin_bit_cast(az_f4, a), y = __builtin_bit_cast(az_f4, b);
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
        return c;
    } else if constexpr (DT == 1)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(az_h8, a), __builtin_bit_cast(az_h8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(az_b8, a), __builtin_bit_cast(az_b8, b), c, 0, 0, 0);
}

// 16-bit rounding to nearest even, and back
template <int DT> __device__ __forceinline__ short az_to16(float x) {
    if constexpr (DT == 1) return __builtin_bit_cast(short, (_Float16)x);
    else return __builtin_bit_cast(short, (__bf16)x);
}
template <int DT> __device__ __forceinline__ float az_from16(short v) {
    if constexpr (DT == 1) return (float)__builtin_bit_cast(_Float16, v);
    else return __uint_as_float((unsigned)(unsigned short)v << 16);
}
// x as hi + lo.  x is fixed to its 32 bits first: where it is a product or a sum of products, the compiler may round it to
// hi in one instruction with them, in another place in two, and lo would then belong to another hi than the one stored.
template <int DT> __device__ __forceinline__ void az_split(float x, short& hi, short& lo) {
    asm("" : "+v"(x));
    hi = az_to16<DT>(x);
    lo = az_to16<DT>(x - az_from16<DT>(hi));
}
// and with a third part: all 24 bits of a bf16 triple
template <int DT> __device__ __forceinline__ void az_split(float x, short& hi, short& lo, short& rest) {
    asm("" : "+v"(x));
    hi = az_to16<DT>(x);
    const float r = x - az_from16<DT>(hi);
    lo = az_to16<DT>(r);
    rest = az_to16<DT>(r - az_from16<DT>(lo));
}
template <int DT> __device__ __forceinline__ float az_load(const void* p, size_t i) {
    if constexpr (DT == 0) return ((const float*)p)[i];
    else return az_from16<DT>(((const short*)p)[i]);
}
template <int DT> __device__ __forceinline__ void az_store(void* p, size_t i, float x) {
    if constexpr (DT == 0) ((float*)p)[i] = x;
    else ((short*)p)[i] = az_to16<DT>(x);
}

// Fragment whose contraction runs along a row of the LDS matrix m [rows][ld]: row r0 + l % 16, elements k0 + EP * (l / 16) ..
template <int DT> __device__ __forceinline__ az_i4 az_row_frag(const void* m, int ld, int r0, int k0, int lane) {
    constexpr int EP = AzElem<DT>::EP, SZ = 16 / EP;
    return *(const az_i4*)((const char*)m + ((r0 + (lane & 15)) * ld + k0 + EP * (lane >> 4)) * SZ);
}
// Fragment whose contraction runs down a column: column n0 + l % 16, rows k0 + EP * (l / 16) ..  For 16-bit elements the
// LDS read transposes: in each group of 16 lanes, lane i's address names 4 elements of row i / 4 and the lane gets
// column i of the 4 x 16 block.  BANKS: group g of lanes takes rows 4 g .. + 3 and 16 more behind, instead of 8 g .. + 7 --
// for products both of whose operands are read this way; with rows an odd multiple of 32 bytes apart the 8 rows of a half
// wave then lie in different banks.
template <int DT, bool BANKS = false> __device__ __forceinline__ az_i4 az_col_frag(const void* m, int ld, int k0, int n0, int lane) {
    if constexpr (DT == 0) {
        const float* p = (const float*)m + (k0 + 4 * (lane >> 4)) * ld + n0 + (lane & 15);
        az_f4 v;
        for (int j = 0; j < 4; ++j) v[j] = p[j * ld];
        return __builtin_bit_cast(az_i4, v);
    } else {
        typedef __attribute__((address_space(3))) az_s4* lds_s4;
        const short* p = (const short*)m + (k0 + (BANKS ? 4 : 8) * (lane >> 4) + ((lane & 15) >> 2)) * ld + n0 + (lane & 3) * 4;
        const az_s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)p);
        const az_s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(p + (BANKS ? 16 : 4) * ld));
        return __builtin_bit_cast(az_i4, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
}

extern "C" int az_internal_fail(int code, const char* msg);          // api.hip: records the message for az_last_error

// A launch on the caller's stream with that stream's device current, the caller's own device put back on every way out.
struct AzDeviceGuard {
    int before = -1;
    bool ok = false;
    explicit AzDeviceGuard(int device) {
        if (hipGetDevice(&before) != hipSuccess) before = -1;
        ok = before == device || hipSetDevice(device) == hipSuccess;
        if (!ok) (void)hipGetLastError();
    }
    ~AzDeviceGuard() { if (before >= 0) (void)hipSetDevice(before); }
};
