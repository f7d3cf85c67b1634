// csrc/devtable.h over the runtime of common.h: a table that `get` hands out is
// written before whatever the caller puts on its stream or into its graph reads it.
#include "devtable.h"

#include <cstdio>

using kfac_devtable::get;
typedef std::vector<std::function<void()>> Graph;

static int failed = 0;
#define CHECK(c) \
  do { if (!(c)) { ++failed; printf("line %d: %s\n", __LINE__, #c); } } while (0)

struct Table {
  char bytes[64];
  explicit Table(int n) { memset(bytes, 0, sizeof(bytes)); memcpy(bytes, &n, sizeof(n)); }
};
static const void* fetch(const Table& t, hipStream_t s) {
  int err = 0;
  const void* p = get(&t, sizeof(t), s, &err);
  CHECK(p && err == 0);
  return p;
}
// a kernel that reads table t through p, on stream s: whether it saw t's bytes
struct Kernel {
  bool ran = false, right = false;
  void launch(const Table& t, const void* p, hipStream_t s) {
    fake::put(s, [this, &t, p] { ran = true; right = p && !memcmp(p, t.bytes, sizeof(t.bytes)); });
  }
};

int main() {
  FakeStream a, b, c;
  {  // one stream, in order; a second fetch costs no copy
    const Table t(1);
    Kernel k1, k2;
    k1.launch(t, fetch(t, &a), &a);
    const int copies = fake::copies;
    k2.launch(t, fetch(t, &a), &a);
    CHECK(fake::copies == copies);
    fake::run(&a);
    CHECK(k1.right && k2.right);
  }
  {  // a second stream does not read before the first one's copy
    const Table t(2);
    Kernel k1, k2;
    k1.launch(t, fetch(t, &a), &a);
    k2.launch(t, fetch(t, &b), &b);
    fake::run(&b);
    CHECK(k2.ran && k2.right);
    fake::run(&a);
    CHECK(k1.right);
  }
  {  // first met in a capture, then called eagerly before the graph runs, then replayed
    const Table t(3);
    Graph g;
    Kernel kg, ke;
    fake::begin(&a, &g);
    kg.launch(t, fetch(t, &a), &a);
    fake::end(&a);
    ke.launch(t, fetch(t, &b), &b);
    fake::run(&b);
    CHECK(ke.ran && ke.right);
    fake::replay(g);
    CHECK(kg.ran && kg.right);
  }
  {  // the capture is abandoned
    const Table t(4);
    Graph g;
    Kernel k;
    fake::begin(&a, &g);
    fetch(t, &a);
    fake::end(&a);
    g.clear();
    k.launch(t, fetch(t, &a), &a);
    fake::run(&a);
    CHECK(k.ran && k.right);
  }
  {  // met in one capture and in another, of which the second runs first
    const Table t(5);
    Graph g, h;
    Kernel k;
    fake::begin(&a, &g);
    fetch(t, &a);
    fake::end(&a);
    fake::begin(&b, &h);
    k.launch(t, fetch(t, &b), &b);
    fake::end(&b);
    fake::replay(h);
    CHECK(k.ran && k.right);
  }
  {  // an eager copy still waits in its stream when a capture meets the table
    const Table t(6);
    Graph g;
    Kernel k, ke;
    ke.launch(t, fetch(t, &a), &a);
    fake::begin(&b, &g);
    k.launch(t, fetch(t, &b), &b);
    fake::end(&b);
    fake::replay(g);
    CHECK(k.ran && k.right);
    fake::run(&a);
    CHECK(ke.right);
  }
  {  // many tables, eager and captured, over several arenas; every one stays what it is
    std::vector<Table> ts;
    std::vector<const void*> ps;
    for (int i = 0; i < 60000; ++i) ts.emplace_back(1000 + i);
    Graph g;
    for (int i = 0; i < 60000; ++i) {
      const bool cap = i % 600 < 500;                     // 500 in a capture, then 100 outside
      if (i % 600 == 0) fake::begin(&a, &g);
      ps.push_back(fetch(ts[i], &a));
      if (i % 600 == 499) fake::end(&a);
      if (!cap && i % 50 == 0) fake::run(&a);
    }
    fake::run(&a);
    int wrong = 0;
    for (int i = 0; i < 60000; ++i) wrong += memcmp(ps[i], ts[i].bytes, sizeof(Table)) != 0;
    CHECK(wrong == 0);
    const int copies = fake::copies;
    for (int i = 0; i < 60000; ++i) CHECK(fetch(ts[i], i & 1 ? &b : &c) == ps[i]);
    CHECK(fake::copies == copies);
    CHECK(fake::allocations > 2);
  }
  CHECK(fake::captures == 0 && fake::forbidden == 0);
  CHECK(fake::mode == hipStreamCaptureModeGlobal);
  CHECK(fake::events < 200);                              // events of ended copies are used again
  printf(failed ? "failed %d\n" : "ok\n", failed);
  return failed != 0;
}
