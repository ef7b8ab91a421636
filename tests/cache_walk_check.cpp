// The heads of a walk (csrc/cache_walk.h): of an append for "append tokens block kv_heads heads threads", of a read for
// "read tokens head_dim kv_heads".
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "cache_walk.h"

int main(int argc, char** argv) {
  const auto n = [&](int i) { return std::atoi(argv[i]); };
  if (argc == 7 && !std::strcmp(argv[1], "append"))
    return std::printf("%d\n", m5k::append_walk(n(2), n(3), n(4), n(5), n(6))), 0;
  if (argc == 5 && !std::strcmp(argv[1], "read")) return std::printf("%d\n", m5k::read_walk(n(2), n(3), n(4))), 0;
  return 1;
}
