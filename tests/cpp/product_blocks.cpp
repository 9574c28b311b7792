// Blocks of a product's results (ProductBlocks): every result in one of them, none of
// more than asked for, the longer side's operand read once where the shorter side fits
// (host only, no GPU). Prints "blocks ok".
#include "cheddar/Transformer.h"

int main() {
  for (int m : {1, 2, 3, 4, 8, 16, 33, 130})
    for (int n : {1, 2, 3, 4, 16, 20, 64, 257})
      for (int results : {1, 2, 3, 5, 10, 64, 128, 1000000}) {
        std::vector<int> seen(m * n, 0);
        int row = 0;
        bool whole_rows = true, whole_cols = true;
        for (const auto &b : cheddar::ProductBlocks(m, n, results)) {
          if (b.i0 >= b.i1 || b.j0 >= b.j1 || b.i0 < row || (b.i1 - b.i0) * (b.j1 - b.j0) > results) return 1;
          row = b.i0;  // rows from the top
          whole_rows &= b.j0 == 0 && b.j1 == n;
          whole_cols &= b.i0 == 0 && b.i1 == m;
          for (int i = b.i0; i < b.i1; i++)
            for (int j = b.j0; j < b.j1; j++) seen[i * n + j]++;
        }
        for (int s : seen)
          if (s != 1) return 2;
        if (results >= m * n && !(whole_rows && whole_cols)) return 3;
        if (m <= n && results >= m && !whole_cols) return 4;
        if (m > n && results >= n && !whole_rows) return 5;
      }
  std::cout << "blocks ok" << std::endl;
  return 0;
}
