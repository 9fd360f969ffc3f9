// Launchers of the paged KV cache's attention kernels (paged.cuh), called by the launchers of their entry points (paged_attn.cu).
#pragma once
#include "paged.cuh"

namespace amv {
namespace paged {

// Maps of the cache for boxes of 64 columns x tokens x heads of one page, and of q for 64 columns x the heads of a group x tokens.
struct Maps {
    CUtensorMap k, v, q;
    bool q_boxes;   // q's map serves the rows of a group
};

constexpr uint32_t kDecRows = 16;                        // paged_attn.cu: rows per tile
constexpr uint32_t kTcRows = 256, kTcKeys = 64;          // paged_tc.cu: rows (half as many for a 32-bit result) and keys per tile

constexpr uint32_t kRenew = 128;                         // key tiles that an accumulator of two row groups takes before it is added to the piece's slot

// exact: one row group, sums added up in registers (32-bit results; also writes f16 ones)
bool launch_tc(const LaunchArgs& a, const Args& pc, const Maps& maps, uint32_t head_dim, uint32_t ctas, bool exact);

}  // namespace paged
}  // namespace amv
