// Copies every shape through alz::CopyCrew and alz::Pieces (audiolazy_amd/csrc/alz_host.h) by way of a small buffer and compares with
// the source; prints "ok <rectangles>" or the first rectangle that differs.  Built and run by tests/test_host_copy_cpu.py.
#include <stdio.h>

#include "../../audiolazy_amd/csrc/alz_host.h"

int main() {
  const size_t widths[] = {1, 8, 63, 64, 65, 200, 511, 512, 513, 4096}, rows[] = {0, 1, 2, 3, 5, 64, 130};
  long n = 0;
  for (int helpers = 0; helpers < 5; ++helpers) {
    alz::CopyCrew crew(helpers);
    for (size_t w : widths)
      for (size_t r : rows)
        for (size_t gap : {(size_t)0, (size_t)24})
          for (size_t cap : {(size_t)200, (size_t)5000}) {
            const size_t sp = w + gap, dp = w + 2 * gap;
            std::vector<char> src(sp * r + 1), dst(dp * r + 1, 7), want(dp * r + 1, 7), buf(cap);
            for (size_t i = 0; i < src.size(); ++i) src[i] = (char)(i * 31 + w);
            for (size_t i = 0; i < r; ++i)
              for (size_t j = 0; j < w; ++j) want[i * dp + j] = src[i * sp + j];
            size_t bytes = 0;
            for (alz::Pieces p(w, r, cap); p.next();) {
              if (p.p_width * p.p_rows > cap || p.p_rows == 0) return printf("a piece of %zu x %zu does not fit %zu\n", p.p_rows, p.p_width, cap), 1;
              crew.copy(buf.data(), p.p_width, src.data() + p.p_row * sp + p.p_col, sp, p.p_width, p.p_rows);
              crew.copy(dst.data() + p.p_row * dp + p.p_col, dp, buf.data(), p.p_width, p.p_width, p.p_rows);
              bytes += p.p_width * p.p_rows;
            }
            if (bytes != w * r || dst != want) return printf("differs: width %zu rows %zu gap %zu buffer %zu helpers %d\n", w, r, gap, cap, helpers), 1;
            ++n;
          }
  }
  printf("ok %ld\n", n);
  return 0;
}
