// policy_loss.hip -- az_policy_loss_dev: argument checks, workspace, launches (the kernels: policy_loss.h)
#include "policy_loss.h"

#include <cstdarg>
#include <cstdio>

namespace {

int lfail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap; va_start(ap, fmt); vsnprintf(buf, sizeof buf, fmt, ap); va_end(ap);
    return az_internal_fail(code, buf);
}

// fp32 weights of more than 32 planes and 128 channels do not fit LDS beside a step: a zero-padded copy [OP][Cp] and one
// transposed [Cp][OP] lie in the workspace, and fragments come from the caches (the fp32 matrix instructions take 32 cycles
// for the 512 bytes of operands that a wave loads).  5 us, a launch.
__global__ void __launch_bounds__(256) az_policy_pad_weight_kernel(const float* w, float* pad, float* padt, int O, int C, int OP, int Cp) {
    for (int i = blockIdx.x * 256 + threadIdx.x; i < OP * Cp; i += gridDim.x * 256) {
        const int o = i / Cp, c = i % Cp;
        const float v = o < O && c < C ? w[(size_t)o * C + c] : 0.f;
        pad[i] = v;
        padt[c * OP + o] = v;
    }
}
// Workgroups' sums added in their order: 64 entries a block, 8 slices of the workgroups.  256 sums of 91 x 129: 12 MB in 4 to
// 5 us, most of it the launch; sums added with atomics would come out in another order each time.
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

hipError_t launch_dt(int dtype, const PolicyDev& a, bool grad, int& groups, hipStream_t stream) {
    if (dtype == AZ_F32) return az_policy_launch_f32(a, grad, groups, stream);
    if (dtype == AZ_F16) return az_policy_launch_f16(a, grad, groups, stream);
    return az_policy_launch_bf16(a, grad, groups, stream);
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
    size_t n = up256((size_t)p->B * sizeof(az_f4));
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
        if (p->counts && p->cap > 1 << 26) return lfail(AZ_E_ARG, "%d targets a board are too many (2^26)", p->cap);   // (times 16 boards: an int)
        const size_t esz = p->dtype == AZ_F32 ? 4 : 2;
        if (((size_t)p->features | (size_t)p->weight | (size_t)p->bias | (size_t)p->d_features) % esz) return lfail(AZ_E_ARG, "a tensor is not aligned to its element type");
        if (((size_t)p->target | (size_t)p->counts | (size_t)p->actions | (size_t)p->probs | (size_t)p->legal | (size_t)p->row_scale | (size_t)p->loss |
             (size_t)p->d_weight | (size_t)p->d_bias) % 4) return lfail(AZ_E_ARG, "a tensor is not aligned to its element type");
    }
    if ((size_t)p->stats % 16) return lfail(AZ_E_ARG, "stats needs 16-byte alignment");
    if (p->B > 0 && grad) {
        // Features, targets and statistics are read while gradients of other boards are written; d_weight and d_bias come last.
        const size_t esz = p->dtype == AZ_F32 ? 4 : 2, B = p->B, cells = (size_t)p->N * p->N, list = B * (p->counts ? p->cap : 0) * 4;
        const struct { const char* name; const void* at; size_t bytes; } in[] = {
            {"features", p->features, B * cells * p->C * esz}, {"weight", p->weight, (size_t)p->c_out * p->C * esz}, {"bias", p->bias, p->c_out * esz},
            {"target", p->target, B * p->c_out * cells * 4}, {"counts", p->counts, B * 4}, {"actions", p->actions, list}, {"probs", p->probs, list},
            {"legal", p->legal, B * p->c_out * p->N * 4}, {"row_scale", p->row_scale, B * 4}, {"stats", p->stats_given ? p->stats : nullptr, B * 16},
        }, out[] = {
            {"d_features", p->d_features, B * cells * p->C * esz}, {"loss", p->loss, B * 4}, {"stats", p->stats_given ? nullptr : p->stats, B * 16},
            {"d_weight", p->d_weight, (size_t)p->c_out * p->C * 4}, {"d_bias", p->d_bias, (size_t)p->c_out * 4},
        };
        const auto meet = [](const auto& a, const auto& b) { return a.at && b.at && (const char*)a.at < (const char*)b.at + b.bytes && (const char*)b.at < (const char*)a.at + a.bytes; };
        for (int i = 0; i < 5; ++i) {
            if (i < 3) for (const auto& x : in) if (meet(out[i], x)) return lfail(AZ_E_ARG, "%s overlaps %s", out[i].name, x.name);
            for (int k = 0; k < i; ++k) if (meet(out[i], out[k])) return lfail(AZ_E_ARG, "%s overlaps %s", out[i].name, out[k].name);
        }
    }
    const size_t need = az_policy_loss_workspace(p);
    if (!workspace) return lfail(AZ_E_ARG, "null argument: workspace");
    if ((size_t)workspace % 256) return lfail(AZ_E_ARG, "workspace needs 256-byte alignment");
    if (workspace_bytes < need) return lfail(AZ_E_CAPACITY, "workspace has %zu bytes, az_policy_loss_workspace asks for %zu", workspace_bytes, need);
    AzDeviceGuard dev(p->device);
    if (!dev.ok) return lfail(AZ_E_HIP, "device %d cannot be used (no HIP device: libazhip has no CPU fallback)", p->device);
    (void)hipGetLastError();                                         // (an earlier call's error is not this one's)
    hipStream_t st = (hipStream_t)stream;
    PolicyDev a = {};
    a.h = p->features; a.w = p->weight; a.bias = p->bias; a.dense = p->target; a.counts = p->counts; a.actions = p->actions; a.probs = p->probs;
    a.legal = p->legal; a.row_scale = p->row_scale; a.scale = p->scale; a.loss = p->loss; a.dh = p->d_features;
    a.B = p->B; a.N = p->N; a.S = p->N * p->N; a.C = p->C; a.O = p->c_out; a.cap = p->cap; a.nchw = p->layout == AZ_CHANNELS_FIRST;
    long long steps;
    geometry(p->B, p->N, a.nb, a.blocks, steps);
    a.steps = (int)steps;
    a.room = a.counts && (long long)a.nb * a.cap <= ENTRIES ? a.nb * a.cap : 0;
    a.mag_n = (65536 + a.N - 1) / a.N; a.mag_s = (65536 + a.S - 1) / a.S; a.mag_w = ((1u << 20) + a.N - 1) / a.N;
    unsigned char* ws = (unsigned char*)workspace;
    a.stats = p->stats ? (az_f4*)p->stats : (az_f4*)ws; ws += up256((size_t)a.B * sizeof(az_f4));
    const bool pads = pads_weight(p);
    float* pad = (float*)ws;
    if (pads) { a.wpad = pad; a.wpadt = pad + PAD_BYTES / 4; ws += 2 * PAD_BYTES; }
    a.partial = (float*)ws;
    int groups = groups_of(a.steps);                                 // (the launch may take fewer)
    hipError_t e = hipSuccess;
    if (a.B > 0 && pads) {
        az_policy_pad_weight_kernel<<<64, 256, 0, st>>>((const float*)p->weight, pad, pad + PAD_BYTES / 4, a.O, a.C, a.O <= 64 ? 64 : a.O <= 96 ? 96 : 128, 256);
        e = hipGetLastError();
    }
    if (e == hipSuccess && a.B > 0 && !p->stats_given) {
        e = launch_dt(p->dtype, a, false, groups, st);
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
