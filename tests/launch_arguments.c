/* Stands in for the HIP runtime, as launch_recorder.c does, and keeps what the library would launch: kernels' names, grids and the first bytes of their first
 * argument.  Loaded ahead of the library with its symbols global, in a process that never loads the runtime proper. */
#include <stdint.h>
#include <string.h>

typedef struct { uint32_t x, y, z; } dim3_t;
enum { kFunctions = 8192, kLaunches = 64, kBytes = 112 };
static struct { const void* f; const char* name; } functions[kFunctions];
static int n_functions = 0;
static struct { const char* name; dim3_t grid, block; unsigned char bytes[kBytes]; } launches[kLaunches];
static int n_launches = 0;
static dim3_t grid_, block_;
static size_t lds_;
static void* stream_;

void** __hipRegisterFatBinary(const void* data) { static void* handle; return (void)data, &handle; }
void __hipUnregisterFatBinary(void** handle) { (void)handle; }
void __hipRegisterFunction(void** handle, const void* f, char* device, const char* name, unsigned limit, void* tid, void* bid, void* bdim, void* gdim, int* wsize) {
  (void)handle, (void)device, (void)limit, (void)tid, (void)bid, (void)bdim, (void)gdim, (void)wsize;
  if (n_functions < kFunctions) functions[n_functions].f = f, functions[n_functions++].name = name;
}
void __hipRegisterVar(void** handle, void* var, char* host, char* device, int ext, size_t size, int constant, int global) {
  (void)handle, (void)var, (void)host, (void)device, (void)ext, (void)size, (void)constant, (void)global;
}
int __hipPushCallConfiguration(dim3_t grid, dim3_t block, size_t lds, void* stream) { return grid_ = grid, block_ = block, lds_ = lds, stream_ = stream, 0; }
int __hipPopCallConfiguration(dim3_t* grid, dim3_t* block, size_t* lds, void** stream) { return *grid = grid_, *block = block_, *lds = lds_, *stream = stream_, 0; }
int hipGetDevice(int* device) { return *device = 0, 0; }
int hipDeviceGetAttribute(int* value, int attribute, int device) { return (void)attribute, (void)device, *value = 256, 0; } /* compute units: all that is asked for */
int hipGetLastError(void) { return 0; }
const char* hipGetErrorString(int e) { return e ? "refused" : "no error"; }
int hipGetSymbolAddress(void** address, const void* symbol) { return *address = (void*)symbol, 0; }
int hipFuncSetAttribute(const void* f, int attribute, int value) { return (void)f, (void)attribute, (void)value, 0; }
int hipLaunchKernel(const void* f, dim3_t grid, dim3_t block, void** args, size_t lds, void* stream) {
  (void)lds, (void)stream;
  if (n_launches == kLaunches) return 1;
  launches[n_launches].name = "";
  for (int i = 0; i < n_functions; ++i)
    if (functions[i].f == f) launches[n_launches].name = functions[i].name;
  launches[n_launches].grid = grid, launches[n_launches].block = block;
  memcpy(launches[n_launches].bytes, args[0], kBytes); /* (an argument on the caller's stack: what follows it is the stack's) */
  return ++n_launches, 0;
}

void recorder_clear(void) { n_launches = 0; }
int recorder_count(void) { return n_launches; }
const char* recorder_name(int i) { return launches[i].name; }
void recorder_get(int i, uint32_t* sizes, unsigned char* bytes) {
  const dim3_t g = launches[i].grid, b = launches[i].block;
  const uint32_t all[6] = {g.x, g.y, g.z, b.x, b.y, b.z};
  memcpy(sizes, all, sizeof(all)), memcpy(bytes, launches[i].bytes, kBytes);
}
