// The host's choice of the layers' tiles, for tests: side and parts of a product, and how a forward product is run.
#include "../gact-icml_amd/csrc/layer_cuts.h"

extern "C" {
// {side, parts, depth of a part}; of codes: a checkpoint's values are one operand
void product_cut(int dtype, int of_codes, int64_t rows, int64_t cols, int64_t depth, int64_t* out) {
  const Cut cut = cut_of(dtype, of_codes, rows, cols, depth, 256, 256);
  out[0] = cut.side;
  out[1] = cut.parts;
  out[2] = cut.per_part;
}
// {few rows, finished, side (rows of a tile that holds codes), parts, depth of a part}
void forward_cut(int dtype, int64_t rows, int64_t inner, int64_t outer, int codes, int whole, int64_t* out) {
  const Forward f = forward_of(dtype, rows, inner, outer, codes, whole);
  out[0] = f.few;
  out[1] = f.finished;
  out[2] = codes && !f.few && !f.finished ? coded_rows_of(dtype == GACT_F32, rows, outer) : f.cut.side;
  out[3] = f.cut.parts;
  out[4] = f.cut.per_part;
}
int compute_units() { return kComputeUnits; }
int workgroups_of_a_unit(int side) { return slots_per_cu(side, side); }
}
