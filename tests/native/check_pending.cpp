// Calls that fail after they have launched kernels, over a runtime that launches nothing and remembers of which stream something is pending: memory that goes
// back to the pools, or to its owner, has nothing pending on it.
#include <hip/hip_runtime_api.h>

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <set>
#include <string>
#include <vector>

#include "../../arboretum_amd/csrc/booster.h"
#include "../../arboretum_amd/csrc/memory_pool.h"
#include "../../arboretum_amd/csrc/operators.h"

#define CHECK(x)                                                    \
  do {                                                              \
    if (!(x)) {                                                     \
      std::printf("%s:%d: %s is false\n", __FILE__, __LINE__, #x);  \
      return 1;                                                     \
    }                                                               \
  } while (0)

namespace {
std::set<hipStream_t> pending;
int launches = 0, fails_at = 0;  // hipGetLastError reports an error once after launch number fails_at
bool failed = false;
std::vector<std::string> given_back_early;
void GiveBack(const char *what) {
  if (!pending.empty()) given_back_early.push_back(what);
}
struct {
  dim3 grid, block;
  size_t lds;
  hipStream_t stream;
} launch;
}  // namespace

extern "C" {
hipError_t hipLaunchKernel(const void *, dim3, dim3, void **, size_t, hipStream_t stream) {
  ++launches;
  pending.insert(stream);
  return hipSuccess;
}
hipError_t hipGetLastError() {
  if (launches != fails_at || failed) return hipSuccess;
  failed = true;
  return hipErrorUnknown;
}
hipError_t hipStreamSynchronize(hipStream_t stream) {
  pending.erase(stream);
  return hipSuccess;
}
hipError_t hipMemcpyAsync(void *, const void *, size_t, hipMemcpyKind, hipStream_t stream) {
  pending.insert(stream);
  return hipSuccess;
}
hipError_t hipMemsetAsync(void *, int, size_t, hipStream_t stream) {
  pending.insert(stream);
  return hipSuccess;
}
hipError_t hipFuncSetAttribute(const void *, hipFuncAttribute, int) { return hipSuccess; }
hipError_t hipStreamWaitEvent(hipStream_t, hipEvent_t, unsigned) { return hipSuccess; }
hipError_t hipEventCreateWithFlags(hipEvent_t *e, unsigned) {
  *e = nullptr;
  return hipSuccess;
}
hipError_t hipEventDestroy(hipEvent_t) { return hipSuccess; }
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }
hipError_t hipEventSynchronize(hipEvent_t) { return hipSuccess; }
const char *hipGetErrorString(hipError_t) { return "an error"; }
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t lds, hipStream_t stream) {
  launch = {grid, block, lds, stream};
  return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3 *grid, dim3 *block, size_t *lds, hipStream_t *stream) {
  *grid = launch.grid;
  *block = launch.block;
  *lds = launch.lds;
  *stream = launch.stream;
  return hipSuccess;
}
void **__hipRegisterFatBinary(const void *) { return nullptr; }
void __hipRegisterFunction(void **, const void *, char *, const char *, unsigned, void *, void *, void *, void *, int *) {}
void __hipUnregisterFatBinary(void **) {}
}

namespace arb {
void *DevicePoolTake(size_t bytes) { return std::malloc(bytes); }
void DevicePoolGive(void *p) noexcept {
  if (p) GiveBack("device memory");
  std::free(p);
}
void *PinnedPoolTake(size_t bytes) { return std::malloc(bytes); }
void PinnedPoolGive(void *p) noexcept {
  if (p) GiveBack("pinned memory");
  std::free(p);
}
hipStream_t StreamPoolTake() { return static_cast<hipStream_t>(std::malloc(1)); }
void StreamPoolGive(hipStream_t s) noexcept {
  if (s) GiveBack("a stream");
  std::free(s);
}

// a matrix whose rows are on the device, or on the host only
static std::vector<float> rows_of_matrix;
static bool rows_on_device;
FloatRows::FloatRows(const float *, size_t n, size_t columns) : n_(n), columns_(columns) {}
FloatRows::~FloatRows() {}
const float *FloatRows::OnHost() { return rows_of_matrix.data(); }
const float *FloatRows::OnDevice() { return rows_on_device ? rows_of_matrix.data() : nullptr; }
DataMatrix::DataMatrix(size_t r, size_t c, size_t cc) : rows(r), columns_dense(c), columns_category(cc), uid(1) {}
DataMatrix::~DataMatrix() {}
std::shared_ptr<const unsigned char> DataMatrix::DeviceLabels() {
  return std::shared_ptr<const unsigned char>(new unsigned char[4](), [](const unsigned char *p) {
    GiveBack("labels");
    delete[] p;
  });
}

static bool log_probs_fail;
size_t LogProbsBytes(long long, long long, int) { return 0; }
void LogProbs(const LogProbsArgs &) {
  if (log_probs_fail) throw std::runtime_error("no");
}
}  // namespace arb

static arb::DataMatrix *Matrix(size_t rows, bool on_device) {
  arb::DataMatrix *m = new arb::DataMatrix(rows, 100, 0);
  m->values.reset(new arb::FloatRows(nullptr, rows, 100));
  arb::rows_of_matrix.assign(rows * 100, 0.0f);
  arb::rows_on_device = on_device;
  return m;
}

// The walk of a matrix fails behind its first launch, or behind a later one of many.
static int Walk() {
  arb::RegTree tree;
  tree.depth = 2;
  tree.fid = {0};
  tree.threshold = {0.5f};
  tree.weights = {1.0f, 2.0f};
  const std::vector<arb::RegTree> trees{tree};
  for (const bool on_device : {true, false})
    for (const int at : {1, on_device ? 1 : 2}) {
      std::unique_ptr<arb::DataMatrix> data(Matrix(on_device ? 1000 : 200000, on_device));
      std::vector<float> sums(data->rows);
      arb::DevicePredictor *p = arb::CreateDevicePredictor();
      launches = 0;
      failed = false;
      fails_at = at;
      bool thrown = false;
      try {
        arb::SumsOnDevice(p, *data, trees, 1, 1, 0.0f, sums.data());
      } catch (const std::runtime_error &) {
        thrown = true;
      }
      CHECK(thrown && launches == at);
      CHECK(pending.empty());  // (the caller gives back `sums`)
      fails_at = 0;
      arb::SumsOnDevice(p, *data, trees, 1, 1, 0.0f, sums.data());
      CHECK(pending.empty());
      arb::FreeDevicePredictor(p);
      for (const std::string &what : given_back_early) std::printf("%s\n", what.c_str());
      CHECK(given_back_early.empty());
    }
  return 0;
}

// Labels are let go once what reads them has ended, also where a later call fails.
static int Labels() {
  for (const bool fails : {false, true}) {
    std::unique_ptr<arb::DataMatrix> data(Matrix(4, true));
    arb::log_probs_fail = fails;
    float sums[8] = {}, log_probs[4];
    bool thrown = false;
    try {
      arb::ClassLogProbsOnDevice(data.get(), sums, 2, arb::ClassLogProbs{0, log_probs, nullptr, nullptr, nullptr});
    } catch (const std::runtime_error &) {
      thrown = true;
    }
    CHECK(thrown == fails && launches == (fails ? 2 : 1));
    for (const std::string &what : given_back_early) std::printf("%s\n", what.c_str());
    CHECK(given_back_early.empty() && pending.empty());
  }
  return 0;
}

int main(int, char **argv) {
  if (!std::strcmp(argv[1], "walk")) return Walk();
  if (!std::strcmp(argv[1], "labels")) return Labels();
  return 2;
}
