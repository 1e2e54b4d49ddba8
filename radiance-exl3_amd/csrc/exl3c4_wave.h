/* exl3c4_wave.h -- what kernels of several files do across a wave's lanes (device code). */
#pragma once

/* The inclusive sum of v over lanes 0 .. lane, by DPP: shifts within each row of 16 lanes, then the rows' totals by row
 * broadcasts (lane 15 into rows 1 and 3, lane 31 into rows 2 and 3). Every lane of the wave must be active. */
static __device__ __forceinline__ int wave_scan_incl(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);   /* row_shr:1 */
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);   /* row_shr:2 */
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);   /* row_shr:4 */
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);   /* row_shr:8 */
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);   /* row_bcast:15 into rows 1, 3 */
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);   /* row_bcast:31 into rows 2, 3 */
    return v;
}
