// Argument blocks and host entry points of the global gradient norm and clipping (clip.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

namespace t2fw {

constexpr int CLIP_TABLE = 144;          // arrays of one launch: the table travels as kernel arguments (4 KB)
constexpr int CLIP_PIECE = 2048;         // elements that are not shared between workgroups: whole vectors for all threads
constexpr int CLIP_GROUPS = 1024;        // workgroups of a launch, at most

struct ClipTable {
    const void *src[CLIP_TABLE];
    void *dst[CLIP_TABLE];
    uint32_t n[CLIP_TABLE];              // elements (longer arrays take several entries)
    uint32_t first[CLIP_TABLE];          // pieces before this array
    uint8_t src_type[CLIP_TABLE], dst_type[CLIP_TABLE];
    int32_t count;
    uint32_t pieces;
};

// sums of squares of a table's arrays, one for each workgroup, to partials[0 .. groups)
int clip_squares(const ClipTable &t, int groups, double *partials, hipStream_t stream);
// norm = sqrt of the sum of all `total` partials; arrays times min(1, max_norm / (norm + 1e-6)), to dst
int clip_scale(const ClipTable &t, int groups, const double *partials, int total, double max_norm, float *norm, hipStream_t stream);

}  // namespace t2fw
