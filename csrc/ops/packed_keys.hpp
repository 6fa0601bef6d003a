// Which keys a row of a tile of packed attention may look through one by one: index arithmetic alone, so that it is tested without a GPU.
#pragma once

namespace mccl {
namespace ops {
namespace packed {

#if defined(__CUDACC__)
#define MCCL_PACKED_FN __host__ __device__ __forceinline__
#else
#define MCCL_PACKED_FN inline
#endif

constexpr int kRows = 128;                 // queries of a tile, and keys of a block

// The keys of block b, from `first` up to but not `end`, of a text with m keys, that a row at position pos does not stand in front of.  A text's last block ends behind its keys,
// and a tile's rows behind its last query have positions behind its last key.
struct BlockKeys {
  int first, end;
};
MCCL_PACKED_FN BlockKeys block_keys(int b, int pos, int m) {
  const int first = b * kRows, last = pos < m - 1 ? pos : m - 1;
  return {first, first + kRows - 1 < last ? first + kRows : last + 1};
}

#undef MCCL_PACKED_FN

}  // namespace packed
}  // namespace ops
}  // namespace mccl
