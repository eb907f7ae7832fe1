// Launch description of the attention kernels, shared by the entry points (rwk_attention.hip) and the instantiations
// per element type (rwk_attention_f32.hip, _f16.hip, _bf16.hip).
#pragma once

#include "rwk_common.h"

struct RwkAttnArgs {
    rwk_attention a;          // as the caller described it
    const int *items;         // a.q_items or a.k_items: segment, first row of the block inside the segment
    int group;                // query heads per key / value head
    int parts, part_heads;    // dK, dV: workgroups that share a block of keys, query heads of each
};

// Which launch of the operator: the forward pass, dQ (which also leaves delta and the partial sums of d_table) or
// dK and dV.
enum RwkAttnPass { kRwkAttnForward, kRwkAttnDq, kRwkAttnDkv };

int rwk_attention_launch_f32(RwkAttnPass pass, const RwkAttnArgs &args, hipStream_t stream);
int rwk_attention_launch_f16(RwkAttnPass pass, const RwkAttnArgs &args, hipStream_t stream);
int rwk_attention_launch_bf16(RwkAttnPass pass, const RwkAttnArgs &args, hipStream_t stream);
