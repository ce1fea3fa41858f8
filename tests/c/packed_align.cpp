// What 4-bit attention's kernels promise of a key piece's address, against the layout: the piece of lane group g at position p of a
// record begins at word 4 p C + g C of keys of C chunks.
#include <attention/attention.hpp>

#include <cstdio>

using namespace certex_amd::attention;

int main()
{
  for (int dim = 1; dim <= 256; ++dim) {
    for (int vdim = 1; vdim <= 256; ++vdim) {
      const int keys = packed_chunks(dim), most = packed_chunks(dim > vdim ? dim : vdim);  // the kernel is of `most`
      const bool full = dim == 32 * most && vdim == 32 * most;
      const int align = packed_key_align(most, full);
      for (int piece = 0; piece < 32; ++piece) {
        if (piece * keys % align != 0) {
          std::printf("%d and %d: piece %d is at word %d, not a multiple of %d\n", dim, vdim, piece, piece * keys, align);
          return 1;
        }
      }
      if (full && align * 4 < 16 && most % 4 == 0) { return 2; }
    }
  }
  std::puts("ok");
  return 0;
}
