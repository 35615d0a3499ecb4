// Argument blocks and host entry points of beam search (beam.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

namespace t2fw {

constexpr int BEAM_COUNT = 128;         // candidates of a call, at most
constexpr int BEAM_ROWS = 256;          // beams of a request, at most

struct BeamArgs {
    const void *logits;                 // [B, K, V] dense
    const float *scores;                // [B, K]
    const uint8_t *finished;            // [B, K] or null
    float *out_scores;                  // [B, n]
    int64_t *out_beams, *out_tokens;    // [B, n]
    void *partial;                      // scratch: [B, K, pieces] largest logits and sums
    uint64_t *lists;                    // scratch: [B, K, pieces, n] best of a piece
    int64_t B, K, V;
    int32_t n, pieces, piece, pad;      // piece: logits of a workgroup
};
struct BeamPieces {
    int32_t pieces, piece;
};
BeamPieces beam_pieces(int64_t B, int64_t K, int64_t V, int64_t n);
int beam_select(const BeamArgs &a, int dtype, hipStream_t stream);

constexpr int REORDER_TABLE = 96;       // arrays of a launch
constexpr int REORDER_BEAMS = 64;       // beams of a request, at most
struct ReorderTable {
    const char *src[REORDER_TABLE];
    char *dst[REORDER_TABLE];
    int64_t row[REORDER_TABLE];         // bytes of one beam
    uint32_t first[REORDER_TABLE];      // the array's first piece of all
    uint32_t count, pieces;
};
int64_t reorder_piece(int64_t K);       // bytes of a beam that a workgroup moves
int beam_reorder(const ReorderTable &t, const int64_t *beams, int64_t B, int64_t K, hipStream_t stream);

}  // namespace t2fw
