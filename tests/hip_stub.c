/* The launch calls of the HIP runtime that a library compiled by hipcc makes, for CPU tests of its host code: kernels are
 * not run, their launches are recorded. A launch that the runtime would refuse (no threads, more than 1024 of them a block, 2^32 or
 * more of them in a dimension) is refused, and so is the one that stub_fail names. Loaded before the library, with its
 * symbols global. */
#include <stdint.h>
#include <stdio.h>
#include <string.h>

typedef struct {
  uint32_t x, y, z;
} dim3_t;
enum { MOST = 100000, KERNELS = 4096 };

static struct {
  const void* at;
  const char* name;
} kernels[KERNELS];
static int n_kernels;

static struct launch {
  const char* name;
  dim3_t grid, block;
  unsigned char first[88]; /* of the kernel's first argument, where its name says that it is a Problem */
} launches[MOST];
static int n_launches, fail_at = -1, fail_with, last_error;

void stub_reset(int at, int with) {
  n_launches = 0;
  fail_at = at;
  fail_with = with;
  last_error = 0;
}
int stub_count(void) { return n_launches; }
const char* stub_name(int i) { return launches[i].name; }
void stub_shape(int i, uint32_t* out) {
  memcpy(out, &launches[i].grid, 12);
  memcpy(out + 3, &launches[i].block, 12);
}
const unsigned char* stub_first(int i) { return launches[i].first; }

void** __hipRegisterFatBinary(const void* data) {
  static void* handle;
  (void)data;
  return &handle;
}
void __hipUnregisterFatBinary(void** modules) { (void)modules; }
void __hipRegisterFunction(void** modules, const void* host, char* device, const char* name, unsigned threads, void* tid, void* bid,
                           void* block, void* grid, int* w) {
  (void)modules, (void)device, (void)threads, (void)tid, (void)bid, (void)block, (void)grid, (void)w;
  if (n_kernels < KERNELS) {
    kernels[n_kernels].at = host;
    kernels[n_kernels++].name = name;
  }
}

static __thread struct {
  dim3_t grid, block;
  size_t shared;
  void* stream;
} pushed;
int __hipPushCallConfiguration(dim3_t grid, dim3_t block, size_t shared, void* stream) {
  pushed.grid = grid;
  pushed.block = block;
  pushed.shared = shared;
  pushed.stream = stream;
  return 0;
}
int __hipPopCallConfiguration(dim3_t* grid, dim3_t* block, size_t* shared, void** stream) {
  *grid = pushed.grid;
  *block = pushed.block;
  *shared = pushed.shared;
  *stream = pushed.stream;
  return 0;
}

int hipLaunchKernel(const void* f, dim3_t grid, dim3_t block, void** args, size_t shared, void* stream) {
  (void)shared, (void)stream;
  struct launch* l = &launches[n_launches < MOST ? n_launches : MOST - 1];
  l->name = "?";
  for (int i = 0; i < n_kernels; ++i)
    if (kernels[i].at == f) l->name = kernels[i].name;
  l->grid = grid;
  l->block = block;
  if (strstr(l->name, "k_product")) memcpy(l->first, args[0], sizeof l->first);
  const int bad = !grid.x || !grid.y || !grid.z || !block.x || !block.y || !block.z || (uint64_t)block.x * block.y * block.z > 1024 ||
                  (uint64_t)grid.x * block.x >> 32 || (uint64_t)grid.y * block.y >> 32 || grid.y > 65535 || grid.z > 65535;
  last_error = n_launches == fail_at ? fail_with : bad ? 9 /* invalid configuration */ : 0;
  if (n_launches < MOST) ++n_launches;
  return last_error;
}
int hipGetLastError(void) {
  const int e = last_error;
  last_error = 0;
  return e;
}
int hipGetDevice(int* d) {
  *d = 0;
  return 0;
}
int hipSetDevice(int d) {
  (void)d;
  return 0;
}
