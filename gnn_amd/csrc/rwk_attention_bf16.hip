// The attention kernels for bf16 rows.
#include "rwk_attention_body.h"

int rwk_attention_launch_bf16(RwkAttnPass pass, const RwkAttnArgs &args, hipStream_t stream) {
    return launch_type<rwk_bf16>(pass, args, stream);
}
