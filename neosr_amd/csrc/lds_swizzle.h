// lds_swizzle.h — where the 16-byte units of a row-major bf16 tile lie in LDS (internal).
//
// The LDS serves 256 bytes (64 banks) a cycle: a ds_read_b128 in phases of 16 lanes, a ds_read_b64_tr_b16 in phases of 32.  MFMA
// operands read the tile in two ways: one unit of 16 consecutive rows (reduction along the row), and 4 units of 4 consecutive
// rows (reduction across rows, transposed on the way).  Unit u of a row is kept at u ^ unit_swizzle(row); both ways then touch
// every 16-byte column of the banks once.  UPR units per row (64-, 128- or 256-byte rows):
//   UPR  4: four rows fill the banks;  rows 4 apart differ in the permutation
//   UPR  8: two rows fill them;        rows 2 apart in bit 2 (another group of 4 units), 4 and 8 apart in bits 0, 1
//   UPR 16: one row fills them;        rows 1, 2 apart in bits 2, 3, rows 4, 8 apart in bits 0, 1
// Period 16 rows.  A permutation for 128-byte phases (rows of 8 lanes) cost twice the LDS cycles (SQ_LDS_BANK_CONFLICT half of
// SQ_LDS_IDX_ACTIVE).
#pragma once
#include <hip/hip_runtime.h>

typedef short s16x4 __attribute__((ext_vector_type(4)));

template <int UPR>
__device__ __forceinline__ int unit_swizzle(int row) {
  static_assert(UPR == 4 || UPR == 8 || UPR == 16, "64-, 128- or 256-byte rows");
  if (UPR == 4) return (row >> 2) & 3;
  if (UPR == 8) return ((row >> 1) & 1) << 2 | ((row >> 2) & 3);
  return (row & 3) << 2 | ((row >> 2) & 3);
}
