// Every 16-byte vector of every row of small matrices at every alignment: whether ends_in_matrix() (csrc/norm.h) lets one through that
// reads behind the matrix's last element.  Prints how many it lets through rightly, wrongly, and holds back without need.
#include <cstdio>

#include "norm.h"

int main() {
  long right = 0, wrong = 0, held = 0;
  for (int vec : {4, 8})
    for (int dim = 1; dim <= 3 * vec; ++dim)
      for (int ld = dim; ld <= dim + vec; ++ld)
        for (int start = 0; start < vec; ++start)
          for (int rows = 1; rows <= 2 * vec; ++rows)
            for (int r = 0; r < rows; ++r) {
              const int first = r * ld, shift = (start + (rows > 1 ? first : 0)) % vec, end = (rows - 1) * ld + dim;
              for (int c = -shift; c < dim; c += vec) {
                const bool inside = first + c + vec <= end;
                if (!rof::ends_in_matrix(r, rows, c, dim, vec)) held += inside && rows - 1 - r >= vec;
                else ++(inside ? right : wrong);
              }
            }
  std::printf("right %ld wrong %ld held %ld\n", right, wrong, held);
  return wrong != 0 || held != 0;
}
