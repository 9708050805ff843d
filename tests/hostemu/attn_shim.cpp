// attn_shim.cpp -- CPU build of the address arithmetic of the cached
// attention kernels (suf_b200/csrc/attention.hpp), so that ragged row
// offsets, bounds and bad pages are checked before any kernel runs.
#include "../../suf_b200/csrc/attention.hpp"

using namespace sufb200;

extern "C" {

int emu_row_len(int n, int L, int causal, int i) { return row_len(n, L, causal, i); }
int64_t emu_row_off(int n, int L, int causal, int i) { return row_off(n, L, causal, i); }

int emu_seq_fits(const sufb200_attn_seqs* s, int c0, int c1, int l0, int l1, int64_t base, int64_t* blk) {
  SeqInfo q;
  const bool ok = seq_fits(*s, c0, c1, l0, l1, base, q);
  *blk = q.blk;
  return ok ? 1 : 0;
}

int64_t emu_page_word(const sufb200_attn_seqs* s, int pg, int kh, int j) { return page_word(*s, pg, kh, j); }

size_t emu_sizeof(int which) { return which == 0 ? sizeof(sufb200_rope_append) : sizeof(sufb200_attn_seqs); }
}

extern "C" int64_t emu_first_block(int64_t c, int b, int per) { return first_block(c, b, per); }
extern "C" int64_t emu_blocks_of(int64_t items, int batch, int per) { return blocks_of(items, batch, per); }
extern "C" int emu_plane_fits(const sufb200_attn_seqs* s, int p0, int p1, int L) { return plane_fits(*s, p0, p1, L); }
