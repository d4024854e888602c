// Copies of operands whose rows are not whole 16 bytes, for the large tiles: rows of whole 16 bytes, zeros behind
// each row's end.  Bound by reading and writing them: a thread moves 16 bytes from any address; the last of a row are
// loaded from where they end with it and shifted.  All operands of a product in one launch: x[1000, 2001] and two
// weights of 4001 rows of bf16 13.4 us (2 x 36 MB: 5.4 TB/s).
#include "projection_common.h"

namespace cmpext3 {
namespace {

__global__ void __launch_bounds__(256) projection_pad_kernel(const PadParams p) {
  const PadParams::Matrix& m = p.m[blockIdx.y];
  const uint32_t pieces = (uint32_t)(m.dst_row / 16);
  const int64_t first = (int64_t)blockIdx.x * 256;
  if (first >= (int64_t)m.rows * pieces) return;
  const int64_t row0 = first / pieces;  // of the workgroup
  const uint32_t at = (uint32_t)(first - row0 * pieces) + threadIdx.x, down = at / pieces;
  const int64_t row = row0 + down;
  if (row >= m.rows) return;
  const int piece = (int)(at - down * pieces);
  const int over = max(16 * piece + 16 - m.row_bytes, 0);  // below 16
  const u32x4 v = *(const u32x4_any*)((const char*)m.src + row * m.src_row + 16 * piece - over);
  *(u32x4*)((char*)m.dst + row * m.dst_row + 16 * piece) = drop_bytes(v, over);
}

}  // namespace

hipError_t launch_projection_pad(const PadParams& p, int count, hipStream_t s) {
  if (count == 0) return hipSuccess;
  int64_t blocks = 0;
  for (int i = 0; i < count; ++i) {
    const int64_t b = ((int64_t)p.m[i].rows * (p.m[i].dst_row / 16) + 255) / 256;
    blocks = b > blocks ? b : blocks;
  }
  if (blocks > UINT32_MAX / 256) return hipErrorInvalidValue;
  return launch_kernel(projection_pad_kernel, dim3((unsigned)blocks, (unsigned)count), dim3(256), 0, s, p);
}

}  // namespace cmpext3
