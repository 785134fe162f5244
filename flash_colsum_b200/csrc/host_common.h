// What the library's translation units share on the host side: error messages, the driver's tensor-map encoder, the
// device's SM count.  Defined in flash_colsum_sm100.cu.
#pragma once

#include <cuda.h>
#include <stdint.h>

namespace fcs {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                  CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                  CUtensorMapFloatOOBfill);

extern thread_local char g_err[512];          // message of the calling thread's last failing call
int fail(int code, const char* fmt, ...);     // stores the message, returns `code`
EncodeTiledFn encode_tiled_fn();              // nullptr where the driver has none
int num_sms();                                // of the current device

// (D, S, H, B) view of a [B, H, S, D] tensor of 16-bit elements, boxes of `box_rows` rows x 64 elements, 128-byte swizzle
int make_tensor_map(CUtensorMap* m, const void* base, int dtype, int B, int H, int S, int D, int64_t sb, int64_t sh,
                    int64_t ss, int box_rows);

}  // namespace fcs
