// Which tiles, and which form of the sums, the logits of the linear head's loss are computed in. Plain C++, no CUDA: the rules of both
// passes stand together because they have to agree.
#pragma once

namespace sx {

constexpr int CE_SEGMENT = 8;  // k-blocks of 64 in a segment of a sum

struct CeTiles {
  int mb;         // row blocks of 128 per CTA of a pair: 1 or 2 (256- and 512-row tiles); 0: single CTAs, up to 128 rows
  bool segments;  // sums of 512 values, joined in registers
  int bn;         // columns of a tile
};

// One CTA up to 128 tokens, else 512-row tiles or 256-row ones: fewer waves x area per tile over the tensor-pipe share
// each shape reaches on large products (0.875 and 0.80, measured for the general pair kernel). The option "pair_mode" (1, 2) decides
// here as it does there.
inline int ce_row_blocks(long long M, long long N, int num_sms, int pair_mode) {
  if (pair_mode == 1 || pair_mode == 2) return pair_mode;
  if (M <= 128) return 0;
  if (M <= 256) return 1;
  const long long pairs = num_sms / 2, nt = (N + 255) / 256;
  const long long w1 = ((M + 255) / 256 * nt + pairs - 1) / pairs, w2 = ((M + 511) / 512 * nt + pairs - 1) / pairs;
  return (double)w2 * 2 / 0.875 <= (double)w1 / 0.80 ? 2 : 1;
}

// Single CTAs: columns of a tile, a multiple of `step` of at most 256, so that every CTA's tiles together have as few columns as can be.
inline int ce_columns_alone(long long N, int step, int least_bn, int num_sms) {
  int best = 256;
  long long least = 1LL << 62;
  for (int bn = 256; bn >= least_bn; bn -= step) {
    const long long tiles = (N + bn - 1) / bn, each = (tiles + num_sms - 1) / num_sms * bn;
    if (each < least) least = each, best = bn;
  }
  return best;
}

// Segments where the error of one sum would be near 1e-6: up to 128 tokens from 2048 values on (1 x 4096 x 65536 101 us, 95
// without), pairs where the sum is longer than 4096 or the vocabulary is small (8192 x 4096 x 50257 would take 2305 us instead of 2164).
// The gradient's logits with them: 2048 x 8192 x 32000 2250 us for the whole pass (2130 without), 300 x 8192 x 8000 192 (188),
// 3 x 8192 x 8205 159 (152).
inline bool ce_in_segments(long long T, long long V, long long H) { return H > 4096 || (H > 2048 && (T <= 128 || V < 16384)); }

// The forward pass. 256-row tiles run in segments whatever the length: one form for them, whose
// epilogue reads a whole accumulator before the lanes' branches (3816 x 1104 x 26330 196 us, 172 as one sum; 200 x 768 x 50257 32, 29;
// 2000 x 256 x 30000, where 512-row tiles are taken, 59, 65).
inline CeTiles ce_forward_tiles(long long T, long long V, long long H, int num_sms, int pair_mode) {
  CeTiles t;
  t.mb = ce_row_blocks(T, V, num_sms, pair_mode);
  t.segments = ce_in_segments(T, V, H);
  if (t.segments && t.mb > 1) t.mb = 1;
  if (t.mb == 1) t.segments = true;
  t.bn = t.mb > 0 ? 256 : ce_columns_alone(V, 16, t.segments ? 64 : 32, num_sms);
  return t;
}

// The gradient, for a piece of n words; `lo`: G in two parts (T <= 64). Its tiles go by the piece, its sums by the forward pass over the whole
// vocabulary. One segment is the same sum in either form. G leaves in blocks of 64 columns.
inline CeTiles ce_gradient_tiles(long long T, long long V, long long H, long long n, bool lo, int num_sms, int pair_mode) {
  CeTiles t;
  t.segments = ce_forward_tiles(T, V, H, num_sms, pair_mode).segments && H > CE_SEGMENT * 64;
  t.mb = lo ? 0 : ce_row_blocks(T, n, num_sms, pair_mode);
  if (t.segments && t.mb > 1) t.mb = 1;
  t.bn = t.mb > 0 ? 256 : ce_columns_alone(n, 64, 64, num_sms);
  return t;
}

// Parts of a row that the forward pass writes, and the most of them whatever the device and the option.
inline int ce_parts(const CeTiles& t, long long V) { return (int)((V + t.bn - 1) / t.bn) * (t.segments || t.mb == 2 ? 2 : 1); }
inline int ce_parts_most(long long T, long long V) {
  const int pairs = (int)((V + 255) / 256) * 2, alone = T <= 128 ? (int)((V + 63) / 64) * 2 : 0;
  return pairs > alone ? pairs : alone;
}

}  // namespace sx
