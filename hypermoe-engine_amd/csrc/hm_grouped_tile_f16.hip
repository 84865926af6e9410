// hm_grouped_tile_f16.hip -- the tile kernels of FP16 operands (hm_grouped_tile.h).
#include "hm_grouped_tile.h"

int hm_g_launch_tiles_f16(GKind kind, int form, bool w_kmajor, bool f32, const GProduct& p, hipStream_t s) {
    return launch_tiles<hm_f16>(form, kind, w_kmajor, f32, p, s);
}
