// The attention kernels for f32 rows.
#include "rwk_attention_body.h"

int rwk_attention_launch_f32(RwkAttnPass pass, const RwkAttnArgs &args, hipStream_t stream) {
    return launch_type<float>(pass, args, stream);
}
