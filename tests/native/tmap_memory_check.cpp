// Host-only check of the TMA descriptor caches (csrc/tmap_cache.h) when memory
// runs out: a descriptor that cannot be kept is still returned, and no exception
// leaves the call (its callers are C entries).  Built and run by
// tests/test_operator_memory_cpu.py with g++; the driver's encoder is a stand-in.
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <new>

#include "tmap_cache.h"

static bool g_full = false;
void* operator new(size_t n) {
  void* p = g_full ? nullptr : std::malloc(n);
  if (!p) throw std::bad_alloc();
  return p;
}
void operator delete(void* p) noexcept { std::free(p); }
void operator delete(void* p, size_t) noexcept { std::free(p); }

static int g_encoded = 0;
static CUresult CUDAAPI encode(CUtensorMap* m, CUtensorMapDataType, cuuint32_t rank, void* ptr, const cuuint64_t*,
                               const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                               CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill) {
  std::memset(m, 0, sizeof(*m));
  std::memcpy(m, &ptr, sizeof(ptr));
  reinterpret_cast<char*>(m)[sizeof(ptr)] = (char)rank;
  ++g_encoded;
  return CUDA_SUCCESS;
}
extern "C" cudaError_t CUDARTAPI cudaGetDriverEntryPoint(const char*, void** fn, unsigned long long,
                                                         cudaDriverEntryPointQueryResult* q) {
  *fn = reinterpret_cast<void*>(&encode);
  *q = cudaDriverEntryPointSuccess;
  return cudaSuccess;
}

template <typename Get, typename Size>
static int check(const char* name, int rank, Get get, Size size) {
  int fails = 0;
  auto expect = [&](bool ok, const char* what) {
    if (!ok) std::printf("%s: %s\n", name, what), ++fails;
  };
  auto is = [&](const CUtensorMap& m, uint64_t ptr) {
    uint64_t p;
    std::memcpy(&p, &m, sizeof(p));
    return p == ptr && reinterpret_cast<const char*>(&m)[sizeof(p)] == (char)rank;
  };
  CUtensorMap m;
  const int before = g_encoded;
  for (bool full : {true, false}) {
    g_full = full;
    try {
      for (uint64_t p = 4096; p <= 8192; p += 4096) {
        std::memset(&m, 0xff, sizeof(m));
        expect(get(p, &m) == 0 && is(m, p), full ? "no descriptor without memory" : "no descriptor");
      }
    } catch (...) {
      expect(false, "an exception left the call");
    }
    g_full = false;
    expect(size() == (full ? 0u : 2u), "entries");
  }
  expect(get(4096, &m) == 0 && is(m, 4096) && g_encoded == before + 4, "a kept descriptor was not reused");
  return fails;
}

int main() {
  pse::TmapCache two;
  pse::Map3Cache three;
  int fails = check("2-D", 2, [&](uint64_t p, CUtensorMap* m) {
    return two.get(reinterpret_cast<void*>(p), 64, 128, 128, 64, 16, 1, m);
  }, [&] { return two.size(); });
  fails += check("3-D", 3, [&](uint64_t p, CUtensorMap* m) {
    return three.get(pse::Map3Key{p, 64, 4, 8, 128, 512, 1, 8}, 1, m);
  }, [&] { return three.size(); });
  std::printf(fails ? "FAIL\n" : "OK\n");
  return fails ? 1 : 0;
}
