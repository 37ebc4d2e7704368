// The kernels of the window attention, chosen between in tpf_window.cu.
#pragma once

#include "tpf_window.cuh"

namespace tpf {

// Few rows over many keys (tpf_window_few.cu): any number of queries, one pass over the keys for every 16 rows.
int window_few(const WindowCall& c, const WindowParams& p, cudaStream_t stream);

// Many queries (tpf_window_fwd.cu): 128 of one head a CTA.
int window_many(const WindowCall& c, const WindowParams& p, cudaStream_t stream);

// Backward (tpf_window_bwd.cu).
int64_t window_bwd_workspace_bytes(const WindowCall& c);
int window_bwd(const WindowCall& c, const WindowParams& p, void* workspace, int64_t workspace_bytes, cudaStream_t stream);

// 4-D map over [B, rows, heads, D] (coordinates: element, row, head, batch) with boxes of 64 elements of `box_rows` rows, 128-byte
// swizzle.  What lies beyond D or the last row comes in as zeros.
int make_window_tmap(CUtensorMap* tm, const void* base, int type, int64_t B, int64_t rows, int64_t heads, int64_t D,
                     const int64_t* strides, int box_rows);

}  // namespace tpf
