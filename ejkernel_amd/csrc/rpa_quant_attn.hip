// Attention over the 8-bit paged cache with block scales: workspace and choice of the instantiation.
#include <algorithm>

#include "rpa_quant_attn.h"

namespace rpa {

namespace {

int padded_dim(const RpaQuantParams& p) { return p.head_dim <= 64 ? 64 : p.head_dim <= 128 ? 128 : 256; }
// Rows of a tile of the second stream: what the instantiation that launch_quant_codes picks has.
int tile_rows(const RpaQuantParams& p) {
  const bool f32 = p.dtype == RPA_DTYPE_F32;
  switch (padded_dim(p)) {
    case 64: return 64 * (f32 ? quant_row_tiles<64, 3>() : quant_row_tiles<64, 1>());
    case 128: return 64 * (f32 ? quant_row_tiles<128, 3>() : quant_row_tiles<128, 1>());
    default: return 64 * (f32 ? quant_row_tiles<256, 3>() : quant_row_tiles<256, 1>());
  }
}
int grid_of() { return std::max(16, 2 * device_cu_count() / 16 * 16); }  // two workgroups per compute unit, the same number on each XCD

struct Layout {
  uint64_t thin_o, thin_ml, tile_o, tile_ml, total;
};
Layout layout(const RpaQuantParams& p, int grid) {
  const uint64_t slots = 2ull * grid, D = padded_dim(p), rows = tile_rows(p);
  Layout l;
  l.thin_o = kWorkspaceTicketBytes;  // the tickets lie in its first kQuantTicketBytes
  l.thin_ml = l.thin_o + slots * 16 * D * 4;
  l.tile_o = l.thin_ml + slots * 16 * 8;
  l.tile_ml = l.tile_o + slots * rows * D * 4;
  l.total = l.tile_ml + slots * rows * 8;
  return l;
}

}  // namespace

uint64_t quant_attention_workspace(const RpaQuantParams& p) { return layout(p, grid_of()).total; }

int launch_quant_attention(const RpaQuantParams& p, hipStream_t stream) {
  QuantArgs a;
  a.p = p;
  a.p.sliding_window = std::min(p.sliding_window, 1 << 30);  // no sequence has more keys, and positions minus a window stay in 32 bits
  a.page_shift = __builtin_ctz(p.page_size);
  a.block_shift = __builtin_ctz(p.scale_block);
  a.group = p.num_q_heads / p.num_kv_heads;
  const int rows = tile_rows(p);
  a.tile_group = std::min(a.group, rows);
  a.tile_tokens = rows / a.tile_group;
  a.subs = (a.group + rows - 1) / rows;
  if (a.subs > 1) a.tile_tokens = 1;
  a.tile_pad = rows > 128 ? 224 : rows > 64 ? 160 : 112;
  a.grid = grid_of();
  int levels = 0;
  while ((1 << levels) < a.grid) ++levels;
  if ((1 + 4ull * levels) * a.grid * sizeof(uint32_t) > kQuantTicketBytes)
    return fail(RPA_ERR_UNSUPPORTED, "a device of %d compute units: the tickets of its workgroups exceed their place", device_cu_count());
  const Layout l = layout(p, a.grid);
  char* ws = static_cast<char*>(p.workspace);
  a.tickets = reinterpret_cast<uint32_t*>(ws);
  a.thin_o = reinterpret_cast<float*>(ws + l.thin_o);
  a.thin_ml = reinterpret_cast<float*>(ws + l.thin_ml);
  a.tile_o = reinterpret_cast<float*>(ws + l.tile_o);
  a.tile_ml = reinterpret_cast<float*>(ws + l.tile_ml);
  switch (code_of_dtype(p.cache_dtype)) {
    case kCodeI8: return launch_quant_i8(a, stream);
    case kCodeE4m3: return launch_quant_e4m3(a, stream);
    default: return launch_quant_e5m2(a, stream);
  }
}

}  // namespace rpa
