/* A CUDA driver and a run-time compiler without a device: the functions that
 * the library binds, over host memory, with kernels run by the SIMT emulator
 * (simt_emul.h).
 *
 * "Compiling" hands the source text on as the machine code;
 * cuModuleGetFunction compiles it for the host with g++ against the emulator's
 * headers. Launches run at once. Every allocation ends at an inaccessible
 * page, so that a read or write beyond it ends the process.
 *
 * SIMT_DIR: the directory of this file, SIMT_TEMPLATES: the kernel templates,
 * SIMT_BUILD: where compiled kernels are kept, SIMT_SMS: multiprocessors. */
#include <cuda.h>
#include <nvrtc.h>
#include <dirent.h>
#include <dlfcn.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <sys/mman.h>
#include <sys/stat.h>
#include <unistd.h>
#include <map>
#include <set>
#include <string>

typedef void (*entry_fn)(void **params, const unsigned *grid, const unsigned *block);
struct fake_module {
  std::string text;
};
static std::map<CUdeviceptr, std::pair<void *, size_t>> blocks;
static int capturing = 0;

static std::string slurp(const std::string &path) {
  std::string s;
  FILE *f = fopen(path.c_str(), "rb");
  if (f == NULL) return s;
  char buf[65536];
  size_t n;
  while ((n = fread(buf, 1, sizeof(buf), f)) > 0) s.append(buf, n);
  fclose(f);
  return s;
}
static std::string env(const char *name) {
  const char *v = getenv(name);
  return v != NULL ? v : "";
}

/* CTAs of a cluster of the kernel: a C expression over the text's macros */
static std::string cluster_of(const std::string &text, const char *kernel) {
  if (strcmp(kernel, "ga_eg_sort_all") == 0) return "GA_EG_CLUSTER";
  if (strcmp(kernel, "ga_lp_rows") == 0) return "GA_LP_CLUSTER";
  return "1";
}

extern "C" {
void fake_cuda_set_capturing(int on) { capturing = on; }

struct _nvrtcProgram {
  std::string text;
};
nvrtcResult nvrtcVersion(int *major, int *minor) { *major = *minor = 0; return NVRTC_SUCCESS; }
const char *nvrtcGetErrorString(nvrtcResult) { return "error"; }
nvrtcResult nvrtcCreateProgram(nvrtcProgram *p, const char *src, const char *, int, const char *const *, const char *const *) {
  *p = new _nvrtcProgram{src};
  return NVRTC_SUCCESS;
}
nvrtcResult nvrtcDestroyProgram(nvrtcProgram *p) { delete *p; return NVRTC_SUCCESS; }
nvrtcResult nvrtcCompileProgram(nvrtcProgram, int, const char *const *) { return NVRTC_SUCCESS; }
nvrtcResult nvrtcGetCUBINSize(nvrtcProgram p, size_t *n) { *n = p->text.size() + 1; return NVRTC_SUCCESS; }
nvrtcResult nvrtcGetCUBIN(nvrtcProgram p, char *out) { memcpy(out, p->text.c_str(), p->text.size() + 1); return NVRTC_SUCCESS; }
nvrtcResult nvrtcGetProgramLogSize(nvrtcProgram, size_t *n) { *n = 0; return NVRTC_SUCCESS; }
nvrtcResult nvrtcGetProgramLog(nvrtcProgram, char *) { return NVRTC_SUCCESS; }

CUresult cuInit(unsigned) { return CUDA_SUCCESS; }
CUresult cuDriverGetVersion(int *v) { *v = 12090; return CUDA_SUCCESS; }
CUresult cuGetErrorName(CUresult, const char **s) { *s = "CUDA_ERROR"; return CUDA_SUCCESS; }
CUresult cuGetErrorString(CUresult, const char **s) { *s = "error"; return CUDA_SUCCESS; }
CUresult cuDeviceGetCount(int *n) { *n = 1; return CUDA_SUCCESS; }
CUresult cuDeviceGet(CUdevice *d, int) { *d = 0; return CUDA_SUCCESS; }
CUresult cuDeviceGetName(char *s, int n, CUdevice) { snprintf(s, n, "emulated"); return CUDA_SUCCESS; }
CUresult cuDeviceGetAttribute(int *v, CUdevice_attribute a, CUdevice) {
  switch (a) {
  case CU_DEVICE_ATTRIBUTE_COMPUTE_CAPABILITY_MAJOR: *v = 10; break;
  case CU_DEVICE_ATTRIBUTE_COMPUTE_CAPABILITY_MINOR: *v = 0; break;
  case CU_DEVICE_ATTRIBUTE_MULTIPROCESSOR_COUNT: *v = atoi(env("SIMT_SMS").c_str()); if (*v <= 0) *v = 2; break;
  case CU_DEVICE_ATTRIBUTE_MAX_SHARED_MEMORY_PER_BLOCK: *v = 49152; break;
  case CU_DEVICE_ATTRIBUTE_MAX_SHARED_MEMORY_PER_BLOCK_OPTIN: *v = 232448; break;
  case CU_DEVICE_ATTRIBUTE_MAX_THREADS_PER_BLOCK: *v = 1024; break;
  case CU_DEVICE_ATTRIBUTE_L2_CACHE_SIZE: *v = 126 << 20; break;
  default: *v = 65535;
  }
  return CUDA_SUCCESS;
}
CUresult cuDeviceTotalMem(size_t *n, CUdevice) { *n = (size_t)1 << 32; return CUDA_SUCCESS; }
CUresult cuDeviceGetPCIBusId(char *s, int n, CUdevice) { snprintf(s, n, "0000:00:00.0"); return CUDA_SUCCESS; }
CUresult cuDevicePrimaryCtxRetain(CUcontext *c, CUdevice) { *c = (CUcontext)1; return CUDA_SUCCESS; }
CUresult cuDevicePrimaryCtxRelease(CUdevice) { return CUDA_SUCCESS; }
CUresult cuCtxPushCurrent(CUcontext) { return CUDA_SUCCESS; }
CUresult cuCtxPopCurrent(CUcontext *c) { *c = (CUcontext)1; return CUDA_SUCCESS; }
CUresult cuCtxGetCurrent(CUcontext *c) { *c = (CUcontext)1; return CUDA_SUCCESS; }
CUresult cuCtxSynchronize(void) { return CUDA_SUCCESS; }
CUresult cuCtxGetDevice(CUdevice *d) { *d = 0; return CUDA_SUCCESS; }
CUresult cuStreamCreate(CUstream *s, unsigned) { *s = (CUstream)2; return CUDA_SUCCESS; }
CUresult cuStreamDestroy(CUstream) { return CUDA_SUCCESS; }
CUresult cuStreamSynchronize(CUstream) { return CUDA_SUCCESS; }
CUresult cuStreamWaitEvent(CUstream, CUevent, unsigned) { return CUDA_SUCCESS; }
CUresult cuStreamIsCapturing(CUstream, CUstreamCaptureStatus *st) {
  *st = capturing ? CU_STREAM_CAPTURE_STATUS_ACTIVE : CU_STREAM_CAPTURE_STATUS_NONE;
  return CUDA_SUCCESS;
}
CUresult cuMemAlloc(CUdeviceptr *p, size_t n) {
  const size_t page = 4096, body = (n + page - 1) / page * page;
  char *m = (char *)mmap(NULL, body + 2 * page, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0);
  if (m == MAP_FAILED) return CUDA_ERROR_OUT_OF_MEMORY;
  mprotect(m, page, PROT_NONE);
  mprotect(m + page + body, page, PROT_NONE);
  memset(m + page, 0xa5, body);
  *p = (CUdeviceptr)(m + page + body - (n + 15) / 16 * 16);
  blocks[*p] = std::make_pair((void *)m, body + 2 * page);
  return CUDA_SUCCESS;
}
CUresult cuMemFree(CUdeviceptr p) {
  munmap(blocks[p].first, blocks[p].second);
  blocks.erase(p);
  return CUDA_SUCCESS;
}
CUresult cuMemHostAlloc(void **p, size_t n, unsigned) { *p = calloc(1, n); return CUDA_SUCCESS; }
CUresult cuMemFreeHost(void *p) { free(p); return CUDA_SUCCESS; }
CUresult cuMemHostGetDevicePointer(CUdeviceptr *d, void *p, unsigned) { *d = (CUdeviceptr)p; return CUDA_SUCCESS; }
CUresult cuMemGetInfo(size_t *f, size_t *t) { *f = *t = (size_t)1 << 32; return CUDA_SUCCESS; }
CUresult cuMemGetAddressRange(CUdeviceptr *, size_t *, CUdeviceptr) { return CUDA_ERROR_NOT_FOUND; }
CUresult cuMemcpyHtoDAsync(CUdeviceptr d, const void *s, size_t n, CUstream) { memcpy((void *)d, s, n); return CUDA_SUCCESS; }
CUresult cuMemcpyDtoHAsync(void *d, CUdeviceptr s, size_t n, CUstream) { memcpy(d, (void *)s, n); return CUDA_SUCCESS; }
CUresult cuMemcpyDtoDAsync(CUdeviceptr d, CUdeviceptr s, size_t n, CUstream) { memmove((void *)d, (void *)s, n); return CUDA_SUCCESS; }
CUresult cuMemcpyPeerAsync(CUdeviceptr d, CUcontext, CUdeviceptr s, CUcontext, size_t n, CUstream) { memmove((void *)d, (void *)s, n); return CUDA_SUCCESS; }
CUresult cuMemsetD8Async(CUdeviceptr d, unsigned char v, size_t n, CUstream) { memset((void *)d, v, n); return CUDA_SUCCESS; }

CUresult cuModuleLoadData(CUmodule *m, const void *image) {
  *m = (CUmodule) new fake_module{std::string((const char *)image)};
  return CUDA_SUCCESS;
}
CUresult cuModuleUnload(CUmodule m) { delete (fake_module *)m; return CUDA_SUCCESS; }
CUresult cuModuleGetFunction(CUfunction *f, CUmodule m, const char *name) {
  const std::string text = ((fake_module *)m)->text +
      "\n#include <type_traits>\n#include <utility>\n"
      "template <class... A, std::size_t... I>\n"
      "static void simt_call(void (*f)(A...), void **p, std::index_sequence<I...>) {\n"
      "  f(*(typename std::remove_cv<A>::type *)p[I]...);\n}\n"
      "template <class... A> static void simt_spread(void (*f)(A...), void **p) {\n"
      "  simt_call(f, p, std::index_sequence_for<A...>());\n}\n"
      "static void simt_body(void *p) { simt_spread(" + std::string(name) + ", (void **)p); }\n"
      "namespace simt { void run_clusters(void (*)(void *), void *, simt_dim3, simt_dim3, unsigned); }\n"
      "extern \"C\" void simt_entry(void **p, const unsigned *g, const unsigned *b) {\n"
      "  const simt_dim3 grid{g[0], g[1], g[2]}, block{b[0], b[1], b[2]};\n"
      "  const unsigned cluster = " + cluster_of(((fake_module *)m)->text, name) + ";\n"
      "  if (cluster > 1) simt::run_clusters(simt_body, p, grid, block, cluster);\n"
      "  else simt::run_grid(simt_body, p, grid, block);\n}\n";
  std::string all = text; /* the key covers every header that the text may include */
  const std::string dirs[2] = {env("SIMT_TEMPLATES"), env("SIMT_DIR") + "/include"};
  for (const std::string &dir : dirs) {
    std::set<std::string> names;
    if (DIR *d = opendir(dir.c_str())) {
      while (dirent *e = readdir(d))
        if (strncmp(e->d_name, "ga_lm", 5) == 0 || strstr(text.c_str(), e->d_name) != NULL ||
            strncmp(e->d_name, "simt", 4) == 0)
          names.insert(e->d_name);
      closedir(d);
    }
    for (const std::string &n : names) all += slurp(dir + "/" + n);
  }
  all += slurp(env("SIMT_DIR") + "/simt_runtime.cpp") + slurp(env("SIMT_DIR") + "/simt_cluster.cpp");
  char key[40];
  snprintf(key, sizeof(key), "%016zx", std::hash<std::string>()(all));
  const std::string base = env("SIMT_BUILD") + "/lm_" + key, so = base + ".so";
  if (access(so.c_str(), R_OK) != 0) {
    mkdir(env("SIMT_BUILD").c_str(), 0777);
    char pid[32];
    snprintf(pid, sizeof(pid), ".%ld", (long)getpid());
    const std::string cpp = base + pid + ".cpp", tmp = base + pid + ".so", log = base + pid + ".log";
    FILE *o = fopen(cpp.c_str(), "wb");
    if (o == NULL) return CUDA_ERROR_FILE_NOT_FOUND;
    fwrite(text.data(), 1, text.size(), o);
    fclose(o);
    const std::string cmd = "g++ -std=c++17 -O1 -shared -fPIC -w -include ga_lm_ptx.cuh -I" + env("SIMT_DIR") + "/include -I" +
                            env("SIMT_TEMPLATES") + " " + cpp + " " + env("SIMT_DIR") +
                            "/simt_runtime.cpp " + env("SIMT_DIR") + "/simt_cluster.cpp -o " + tmp + " > " + log + " 2>&1";
    if (system(cmd.c_str()) != 0) {
      fprintf(stderr, "%s\n%s\n", cmd.c_str(), slurp(log).substr(0, 4000).c_str());
      return CUDA_ERROR_INVALID_SOURCE;
    }
    rename(tmp.c_str(), so.c_str());
    unlink(cpp.c_str());
    unlink(log.c_str());
  }
  void *h = dlopen(so.c_str(), RTLD_NOW | RTLD_LOCAL);
  if (h == NULL) {
    fprintf(stderr, "%s\n", dlerror());
    return CUDA_ERROR_INVALID_SOURCE;
  }
  *f = (CUfunction)dlsym(h, "simt_entry");
  return *f != NULL ? CUDA_SUCCESS : CUDA_ERROR_NOT_FOUND;
}
CUresult cuFuncGetAttribute(int *v, CUfunction_attribute a, CUfunction) {
  *v = a == CU_FUNC_ATTRIBUTE_MAX_THREADS_PER_BLOCK ? 1024 : 32;
  return CUDA_SUCCESS;
}
CUresult cuFuncSetAttribute(CUfunction, CUfunction_attribute, int) { return CUDA_SUCCESS; }
CUresult cuLaunchKernel(CUfunction f, unsigned gx, unsigned gy, unsigned gz, unsigned bx, unsigned by,
                        unsigned bz, unsigned, CUstream, void **params, void **) {
  const unsigned g[3] = {gx, gy, gz}, b[3] = {bx, by, bz};
  if (gx == 0 || gy == 0 || gz == 0 || gy > 65535 || bx * by * bz == 0 || bx * by * bz > 1024)
    return CUDA_ERROR_INVALID_VALUE;
  ((entry_fn)f)(params, g, b);
  return CUDA_SUCCESS;
}
CUresult cuLaunchKernelEx(const CUlaunchConfig *c, CUfunction f, void **params, void **extra) {
  return cuLaunchKernel(f, c->gridDimX, c->gridDimY, c->gridDimZ, c->blockDimX, c->blockDimY, c->blockDimZ,
                        c->sharedMemBytes, c->hStream, params, extra);
}
CUresult cuOccupancyMaxActiveBlocksPerMultiprocessor(int *n, CUfunction, int, size_t) { *n = 4; return CUDA_SUCCESS; }
CUresult cuEventCreate(CUevent *e, unsigned) { *e = (CUevent)3; return CUDA_SUCCESS; }
CUresult cuEventRecord(CUevent, CUstream) { return CUDA_SUCCESS; }
CUresult cuEventSynchronize(CUevent) { return CUDA_SUCCESS; }
CUresult cuEventElapsedTime(float *t, CUevent, CUevent) { *t = 0; return CUDA_SUCCESS; }
CUresult cuEventDestroy(CUevent) { return CUDA_SUCCESS; }
CUresult cuIpcGetMemHandle(CUipcMemHandle *, CUdeviceptr) { return CUDA_ERROR_NOT_SUPPORTED; }
CUresult cuIpcOpenMemHandle(CUdeviceptr *, CUipcMemHandle, unsigned) { return CUDA_ERROR_NOT_SUPPORTED; }
CUresult cuIpcCloseMemHandle(CUdeviceptr) { return CUDA_ERROR_NOT_SUPPORTED; }
}
