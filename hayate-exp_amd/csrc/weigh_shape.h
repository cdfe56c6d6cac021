// Shape of the work items that add up attention weights, shared by the planner (host) and the
// kernels.
#pragma once

namespace hy {

// Keys of one item: four waves of 64.
constexpr int kWeighKeys = 256;
// Query rows (token, head) of one load stage.
constexpr int kWeighRows = 64;
// Scores of a sequence's decode token start at a multiple of this (whole slices of the decode
// kernel are stored).
constexpr int kWeighPad = 32;

}  // namespace hy
