// policy_loss.h -- cross entropy of the policy head (PolicyHead's 1x1 convolution and its softmax over all
// c_out * N * N entries, network.hpp:46-65; the policy term of the trainer's loss, train.cpp:90-112) with its gradients,
// without the logits ever being written.
//
//   z[b,o,s]  = sum_c w[o,c] h[b,c,s] + bias[o]                      s = cell of the board, S = N * N
//   lse_b     = log sum over the allowed (o, s) of exp z             loss_b = sum_{t != 0} t (lse_b - z)
//   dz[b,o,s] = r_b (T_b exp(z - lse_b) - t) on allowed entries, 0 elsewhere;  T_b = sum t
//   dh = w^T dz      dw = sum dz h^T      dbias = sum dz
//
// Rows of the work are the cells of boards, 16 to a tile.  az_policy_loss_kernel takes a whole board a workgroup (several
// where they are small, 32 cells or fewer), forms its logits in registers and keeps a running {max, sum of exp, sum t z,
// sum t} over them.  az_policy_grad_kernel forms the same logits again, 64 rows a step -- 2 C flop an entry against 8 bytes
// of a kept fp32 logit written and read -- turns them into dz in LDS and multiplies it both ways; az_policy_reduce_kernel
// adds the workgroups' dw and dbias in a fixed order.
//
// The features are read twice, once for the losses and once for the gradients: a board's lse is not known before all of its
// logits are.  Times are those of an MI355X that copies 4.9 TB/s and multiplies 1.1 PFLOP/s (16 bits) / 154 TFLOP/s (fp32).
#pragma once
#include "../../include/az_hip.h"
#include "az_learn.h"

constexpr int ROWS = 64;                     // rows of a step
constexpr size_t LDS_BYTES = 160 * 1024;
constexpr int CUS = 256, NT = 512, WAVES = 8;
constexpr int MAX_GROUPS = 512;              // workgroups of the gradient kernel: two a CU
constexpr int ENTRIES = 2 * NT;              // sparse targets of a workgroup's boards kept in LDS; longer lists are read from memory
constexpr int MAX_BOARDS = 16;               // boards of a workgroup
constexpr float LOG2E = 1.4426950408889634f;

struct PolicyDev {
    const void *h, *w, *bias;
    const float* dense;                      // [B, O * S] or null
    const int *counts, *actions;             // [B], [B, cap]
    const float* probs;                      // [B, cap]
    const unsigned* legal;                   // [B, O * N] or null
    const float* row_scale;                  // [B] or null
    float scale;
    az_f4* stats;                            // [B] {max z, T, 1 / sum of exp(z - max), fp16: sum |t|, other types: 1}; the last negative
                                             // where a target outside the allowed actions makes the loss infinite
    float *loss, *partial;
    const float *wpad, *wpadt;               // fp32 weights that do not fit LDS: padded copies
    void* dh;
    int B, N, S, C, O, cap, nchw;
    int room;                                // sparse targets that LDS has room for: those of a workgroup's boards, or 0 = read from memory
    int nb, blocks;                          // boards a workgroup takes at once (blocks = 1), or steps a board is cut into (nb = 1)
    int steps;                               // of the gradient kernel
    unsigned mag_n, mag_s, mag_w;            // x / N = x * mag_n >> 16 for x < 1024 = x * mag_w >> 20 for x < 4096, x / S = x * mag_s >> 16 for x < 64
};

// the two product kernels of one element type (policy_f32.hip, policy_f16.hip, policy_bf16.hip)
hipError_t az_policy_launch_f32(const PolicyDev& a, bool grad, int& groups, hipStream_t stream);
hipError_t az_policy_launch_f16(const PolicyDev& a, bool grad, int& groups, hipStream_t stream);
hipError_t az_policy_launch_bf16(const PolicyDev& a, bool grad, int& groups, hipStream_t stream);
