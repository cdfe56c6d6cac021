// Shape of a drafted-tree attention work item, shared by the planner (host) and
// the kernel: the work lists and the split workspace are laid out by it.
#pragma once

namespace hy {

// (node, head) rows of one workgroup at most: eight waves of 32.
constexpr int kTreeRows = 256;
// Keys per step; a piece's keys start at a multiple of it.
constexpr int kTreeTileKeys = 64;
// Nodes of one tree at most (a node's ancestors are a mask of 32-bit words).
constexpr int kTreeMaxNodes = 256;
// 32-bit fields of a chunk record: the chunk's own eight, then its first piece.
constexpr int kTreeChunkInts = 16;

}  // namespace hy
