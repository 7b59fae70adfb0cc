// guard_alloc.cpp -- a torch.cuda pluggable allocator that puts an UNMAPPED guard range right behind every tensor (debugging aid).
// Each allocation is its own virtual-memory reservation: `size` rounded up to the mapping granularity is backed
// by physical memory, one more granule behind it is reserved and never mapped, and the tensor is placed so that it ENDS at the
// end of the mapped range (start 16-byte aligned: at most 15 bytes of slack).  A kernel that reads or writes 16 bytes past the end
// of any buffer takes a GPU memory fault at that very launch -- whatever the caching allocator's layout would have hidden.
//   hipcc -O2 -shared -fPIC -o /tmp/libguard_alloc.so tools/dbg/guard_alloc.cpp
//   FDGAN_TEST_GUARD_ALLOC=/tmp/libguard_alloc.so python -m pytest tests -m gpu ...   (tests/conftest.py)
#include <hip/hip_runtime.h>
#include <stdio.h>
#include <stdlib.h>
#include <sys/types.h>

#include <mutex>
#include <unordered_map>

namespace {
struct Rec {
  void* va;
  size_t mapped, reserved;
  hipMemGenericAllocationHandle_t h;
};
std::mutex g_mu;
std::unordered_map<void*, Rec> g_live;
size_t g_gran = 0;
long long g_allocs = 0, g_bytes = 0;

#define GCHK(x)                                                                                   \
  do {                                                                                            \
    hipError_t e_ = (x);                                                                          \
    if (e_ != hipSuccess) {                                                                       \
      fprintf(stderr, "[guard_alloc] %s failed: %s (size %zu)\n", #x, hipGetErrorString(e_), (size_t)size); \
      abort();                                                                                    \
    }                                                                                             \
  } while (0)
}  // namespace

// Where a tensor of `size` bytes lies: returns its offset in the mapped range, whose length goes to `mapped` (whole granules).  At the end
// (16-byte aligned: at most 15 bytes of slack) or at the start.
extern "C" size_t guard_place(size_t size, size_t gran, int at_end, size_t* mapped) {
  *mapped = (size + gran - 1) / gran * gran;
  return at_end ? (*mapped - size) & ~(size_t)15 : 0;
}

extern "C" void* guard_malloc(ssize_t size, int device, hipStream_t stream) {
  if (size <= 0) return nullptr;
  std::lock_guard<std::mutex> lk(g_mu);
  hipMemAllocationProp prop = {};
  prop.type = hipMemAllocationTypePinned;
  prop.location.type = hipMemLocationTypeDevice;
  prop.location.id = device;
  if (g_gran == 0) {
    GCHK(hipMemGetAllocationGranularity(&g_gran, &prop, hipMemAllocationGranularityMinimum));
    fprintf(stderr, "[guard_alloc] granularity %zu bytes\n", g_gran);
  }
  // GUARD_ALLOC_END=1: the tensor ENDS at the guard (start only 16-byte aligned).  torch's own fills / copies then leave the tail of such
  // tensors unwritten unless nothing is ever unmapped (GUARD_ALLOC_LEAK=1; results wrong, no fault), so the default places the tensor
  // at the START of its page-aligned mapping: tensors whose size is a multiple of the 4 KiB granule -- every large power-of-two activation /
  // gradient buffer, exactly the ones that end at a segment boundary under the caching allocator -- still end exactly at the guard.
  static const bool at_end = getenv("GUARD_ALLOC_END") != nullptr;
  Rec r;
  const size_t offset = guard_place((size_t)size, g_gran, at_end, &r.mapped);
  r.reserved = r.mapped + g_gran;
  GCHK(hipMemAddressReserve(&r.va, r.reserved, g_gran, nullptr, 0));
  GCHK(hipMemCreate(&r.h, r.mapped, &prop, 0));
  GCHK(hipMemMap(r.va, r.mapped, 0, r.h, 0));
  hipMemAccessDesc acc = {};
  acc.location = prop.location;
  acc.flags = hipMemAccessFlagsProtReadWrite;
  GCHK(hipMemSetAccess(r.va, r.mapped, &acc, 1));
  char* p = static_cast<char*>(r.va) + offset;
  g_live[p] = r;
  ++g_allocs, g_bytes += r.mapped;
  return p;
}

extern "C" void guard_free(void* ptr, ssize_t size, int device, hipStream_t stream) {
  if (ptr == nullptr) return;
  (void)hipDeviceSynchronize();      // nothing may still be using it (this allocator knows nothing about streams)
  std::lock_guard<std::mutex> lk(g_mu);
  auto it = g_live.find(ptr);
  if (it == g_live.end()) {
    fprintf(stderr, "[guard_alloc] free of an unknown pointer %p\n", ptr);
    return;
  }
  Rec r = it->second;
  g_live.erase(it);
  static const bool leak = getenv("GUARD_ALLOC_LEAK") != nullptr;      // never unmap (isolates "freed too early" from "read past the end")
  if (leak) return;
  (void)hipMemUnmap(r.va, r.mapped);
  (void)hipMemRelease(r.h);
  (void)hipMemAddressFree(r.va, r.reserved);
}
