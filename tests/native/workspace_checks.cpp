// Checks of csrc/device_cache.h's workspaces that are given up, over a fake backend
// (malloc), built with sanitizers by tests/test_workspace.py.  Exit status 0 = all
// checks passed.
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "device_cache.h"

using namespace tt;

static int g_failures = 0;
#define CHECK(cond)                                                           \
  do {                                                                        \
    if (!(cond)) {                                                            \
      std::fprintf(stderr, "CHECK failed at line %d: %s\n", __LINE__, #cond); \
      ++g_failures;                                                           \
    }                                                                         \
  } while (0)

struct FakeBackend {
  long syncs = 0;
  int sync_fails = 0;
  int alloc(size_t bytes, void** p) {
    *p = std::malloc(bytes);
    return *p ? 0 : 4;
  }
  void release(void* p) { std::free(p); }
  int sync(void*) {
    ++syncs;
    return sync_fails;
  }
  int order_after_library(void*) { return 0; }
};

int main() {
  FakeBackend be;
  BlockCache<FakeBackend> blocks(be);
  WorkspaceCache<FakeBackend> ws(be, blocks);
  int s1 = 0, s2 = 0;
  void *p = nullptr, *q = nullptr, *lost = nullptr;
  uint64_t uses = 99;
  size_t used = 0;
  {
    WorkspaceCache<FakeBackend>::Lease l(ws);
    CHECK(l.get(&s1, 0, 4096, &p, &uses) == 0 && uses == 0);
    CHECK(l.get(&s1, 1, 64, &q) == 0 && l.get(&s2, 0, 64, &q) == 0);
    l.drop(&s1, 0);  // waits, and the buffer is there no more
    CHECK(be.syncs == 1);
    CHECK(!l.get_held(&s1, 0, 1, &q) && l.get_held(&s1, 1, 64, &q) && l.get_held(&s2, 0, 64, &q));
    l.drop(&s1, 0);  // nothing to give up
    l.drop(&s2, 7);
    CHECK(be.syncs == 1);
  }
  CHECK(ws.count() == 2);
  {
    WorkspaceCache<FakeBackend>::Lease l(ws);
    uses = 99;
    CHECK(l.get(&s1, 0, 4096, &q, &uses) == 0 && uses == 0);  // new to its user, though the block may be the old one
    std::memset(q, 1, 4096);
    CHECK(l.get(&s1, 0, 4096, &q, &uses) == 0 && uses == 1);
    lost = q;
    be.sync_fails = 3;
    l.drop(&s1, 0);  // work may still use the block: nobody gets it
    be.sync_fails = 0;
    CHECK(l.get(&s1, 0, 4096, &q, &uses) == 0 && uses == 0 && q != lost);
  }
  CHECK(ws.release_all() == 0);
  blocks.trim();
  blocks.stats(&used, nullptr);
  CHECK(used == 4096);  // the lost one
  blocks.release(lost);
  blocks.trim();
  if (g_failures) return 1;
  std::puts("workspace checks passed");
  return 0;
}
