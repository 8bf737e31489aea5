/* The stream's workspace, shared by the serving kernels: the kernels of a stream run one after the
 * other, and each leaves the counters at zero. */
#ifndef SERVE_WS_H_
#define SERVE_WS_H_

#include "glint_common.h"

/* As glint_split_ws_stream (tile_mfma.h); one cache for the library. */
bool glint_serve_ws(hipStream_t stream, GlintSplitWs &ws);

#endif
