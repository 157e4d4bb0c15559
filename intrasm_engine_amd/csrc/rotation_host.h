// A rotation's arguments, checked, as the kernels take it.
#pragma once
#include "paged_cache_host.h"
#include "rotation_device.cuh"

namespace iex {
namespace {

// Of a call that has tokens.  Null `at`: the caller knows where they are, and that the table has those rows.
int check_rotation(const iex_rotation* r, const char* what, Rotation& out) {
  out = Rotation{};
  out.axes = 1;
  if (!r || r->features == 0) {
    IEX_REQUIRE(!r || !r->at, IEX_ERR_BAD_ARGUMENT, "%s: positions without a rotation", what);
    return 0;
  }
  IEX_REQUIRE(r->features > 0 && r->rows >= 0, IEX_ERR_BAD_ARGUMENT, "%s: negative dimension", what);
  IEX_REQUIRE(r->table && aligned(r->table, 16), IEX_ERR_BAD_ARGUMENT, "%s: the rotation must be a 16-byte aligned array", what);
  out.table = r->table, out.rows = r->rows, out.features = r->features;
  if (!r->at) {
    IEX_REQUIRE(r->axes <= 1 && !r->sections, IEX_ERR_BAD_ARGUMENT, "%s: several axes without positions", what);
    return 0;
  }
  IEX_REQUIRE(r->rows > 0, IEX_ERR_BAD_ARGUMENT, "%s: the rotation must have a row", what);
  IEX_REQUIRE(r->axes >= 1 && r->axes <= 4, IEX_ERR_UNSUPPORTED, "%s: positions of one to four axes (%d)", what, r->axes);
  IEX_REQUIRE(aligned(r->at, 4), IEX_ERR_UNSUPPORTED, "%s: operands must be aligned to their elements", what);
  out.positions = r->at, out.axis_stride = r->axis_stride, out.axes = r->axes;
  if (r->axes == 1 && !r->sections) return 0;
  IEX_REQUIRE(r->sections, IEX_ERR_BAD_ARGUMENT, "%s: positions of several axes need sections", what);
  IEX_REQUIRE(r->features <= 256, IEX_ERR_UNSUPPORTED, "%s: up to 256 rotated features by sections (%d)", what, r->features);
  int left[4] = {0, 0, 0, 0}, total = 0;
  for (int a = 0; a < r->axes; ++a) {
    IEX_REQUIRE(r->sections[a] >= 0 && r->sections[a] <= 128, IEX_ERR_BAD_ARGUMENT, "%s: a section of %d planes", what, r->sections[a]);
    total += left[a] = r->sections[a];
  }
  IEX_REQUIRE(2 * total == r->features, IEX_ERR_BAD_ARGUMENT, "%s: sections of %d planes, the rotation has %d", what, total, r->features / 2);
  for (int plane = 0, axis = 0; plane < total; ++plane) {
    while (left[axis] == 0) axis = (axis + 1) % r->axes;
    out.axis_of[plane / 32] |= (unsigned long long)axis << (plane % 32 * 2);
    --left[axis];
    if (r->in_turn) axis = (axis + 1) % r->axes;
  }
  return 0;
}

}  // namespace
}  // namespace iex
