// Declarations shared by the host side (packed.cpp) and the kernels
// (packed.hip, attention_masked.hip) of the operators on packed documents.
#pragma once

#include <hip/hip_runtime_api.h>

#include <cstdint>

namespace svl {

// A segment of a position plan: a text run (area 0) or a grid of rows of
// `cols` tokens, `area` tokens a frame, `step` positions apart.
struct PositionSegment {
    int32_t begin;  // first token
    int32_t start;  // position of the segment's first token
    int32_t area, cols, step;
};
constexpr int POSITION_BLOCK = 1024;  // tokens per workgroup

// block_seg[b]: the segment that token b * POSITION_BLOCK lies in (one more
// entry at the end: the last segment).
hipError_t launch_axis_positions(const PositionSegment *seg, const int32_t *block_seg,
                                 int64_t tokens, int32_t *pos, hipStream_t s);

constexpr int ROPE_MAX_PAIRS = 256;

struct RopeAxesArgs {
    const void *in[2];
    void *out[2];
    int64_t in_tok[2], in_head[2], out_tok[2], out_head[2];
    int32_t heads[2];
    const int32_t *pos;
    int64_t tokens;
    int32_t axes, hd, pairs, copied;  // copied: columns past the pairs that go to `out`
    float inv_freq[ROPE_MAX_PAIRS];
    uint16_t col[ROPE_MAX_PAIRS];      // first column of each pair
    uint16_t partner[ROPE_MAX_PAIRS];  // its other column
    uint8_t axis[ROPE_MAX_PAIRS];
};
// ROPE_CHUNKS: pairs in runs of whole 16-byte chunks in both columns (adjacent:
// in one), every row at a multiple of 16 bytes; ROPE_ROWS: rows of whole chunks
// at such addresses; ROPE_SINGLE: any.
enum RopeForm { ROPE_CHUNKS, ROPE_ROWS, ROPE_SINGLE };
hipError_t launch_rope_axes(const RopeAxesArgs &a, bool bf16, bool adjacent, RopeForm form,
                            hipStream_t s);

// One workgroup's work in masked attention: query vectors v0 .. of one
// document and KV head (vector v is query v / G, head kvh * G + v % G, G heads
// per KV head) against key tiles t0 .. t1 of its tile list. The list is
// pre_tiles tiles from key 0 (they cover the prefix), then tiles from key
// main_key on.
struct AttnWork {
    int32_t q_row, q_len, k_row, k_len;  // the document's rows
    int32_t kvh, v0;
    int32_t prefix;
    int32_t pre_tiles, main_key;
    int32_t t0, t1;
    int32_t slot;   // partial result's place in the workspace, -1: to the output
    int32_t tile0;  // first of the document and KV head's tiles of planes
};
// A tile of planes: keys from row k_row on, `rows` of them.
struct AttnTiles {
    int32_t k_row, rows, kvh;
};
// A group of vectors whose key tiles were split over `parts` workgroups.
struct AttnJoin {
    int32_t q_row, q_len, kvh, v0, slot, parts;
};

constexpr int MASKED_MOST_PARTS = 1280;  // of one group

struct MaskedArgs {
    const void *q, *k, *v;
    void *out;
    float *lse;
    int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head;
    int32_t heads, kv_heads, hd;
    int32_t causal, window;  // window < 0: none
    float scale, cap;
    const float *slopes;
    const AttnWork *work;
    int32_t n_work;
    const AttnJoin *join;
    int32_t n_join, join_vectors, join_parts;  // most vectors and parts of a joined group
    float *partial;
    void *planes;  // tiles of keys and values, where the shape has them
    const AttnTiles *tiles;
    int32_t n_tiles;
    int32_t whole;   // every row in whole 16-byte chunks at 16-byte addresses
};

// The kernel that a plan is made for, and its tiles.
struct MaskedShape {
    int dim;      // head dim that its tiles hold, 0: the kernel of one wave a query
    int vectors;  // query vectors per workgroup
    int keys;     // keys per tile
    int planes;   // parts that keys and values are split into before, 0: none
    int slots;    // workgroups that the GPU holds at once
    int least;    // key tiles that are worth a workgroup of their own
};
// most: query vectors of the batch's largest document and KV head.
MaskedShape masked_shape(bool bf16, int hd, int64_t most);
// Floats of a slot of the workspace: outputs, maxima and sums of its vectors, in
// whole 16 bytes.
constexpr int64_t masked_slot(int vectors, int dim) {
    return ((int64_t)vectors * (dim + 2) + 3) / 4 * 4;
}
// Bytes of a tile of planes: keys and values.
inline int64_t masked_tile_bytes(const MaskedShape &s) {
    return (int64_t)2 * s.planes * s.keys * s.dim * 2;
}
hipError_t launch_masked_attention(MaskedArgs a, bool bf16, const MaskedShape &shape,
                                   hipStream_t s);

}  // namespace svl
