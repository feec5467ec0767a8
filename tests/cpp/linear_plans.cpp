// Prints the plans that the mixed-precision product chooses. Each line of input is a call:
//   products vec M N K [M N K]      (one or two products, the one with more k first)
// and each line of output its launches:  products qc bn cg split [products qc bn cg split]
#include <cstdio>
#include <cstring>

#include "../../paralia-framework_b200/csrc/gemm_act_plan.hpp"

int main() {
  int n = 0, vec = 0;
  while (scanf("%d %d", &n, &vec) == 2 && n >= 1 && n <= 2) {
    paralia::GemmActProblem p[2];
    memset(p, 0, sizeof(p));
    for (int i = 0; i < n; ++i)
      if (scanf("%d %d %d", &p[i].M, &p[i].N, &p[i].K) != 3) return 1;
    paralia::GaPlan plans[2];
    const int launches = paralia::ga_plan_launches(p, n, vec != 0, plans);
    for (int i = 0; i < launches; ++i)
      printf("%s%d %d %d %d %d", i ? " " : "", launches == 1 ? n : 1, (int)plans[i].qc, plans[i].bn, plans[i].cg, plans[i].split);
    printf("\n");
  }
  return 0;
}
