// The attention kernels for f16 rows.
#include "rwk_attention_body.h"

int rwk_attention_launch_f16(RwkAttnPass pass, const RwkAttnArgs &args, hipStream_t stream) {
    return launch_type<rwk_f16>(pass, args, stream);
}
