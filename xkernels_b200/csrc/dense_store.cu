// Dense products that are stored as they are (dense_dev.cuh).
#include "dense_dev.cuh"

namespace xkb {
namespace dense {

int run_store(bool b_mn, const Params& p, const Launch& l) {
  return b_mn ? run_variant<true, kStore>(p, l) : run_variant<false, kStore>(p, l);
}

}  // namespace dense
}  // namespace xkb
