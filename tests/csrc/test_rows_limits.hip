// The templates between tokens and rows throw hipErrorInvalidValue for sizes
// that their kernels cannot index, before they allocate or launch anything:
// through a context that does neither, so this runs without a GPU.
// Exit status 1 if a call does something else.
#include <moderngpu/kernel_embedding.hxx>
#include <moderngpu/kernel_distill.hxx>
#include <moderngpu/kernel_sample.hxx>
#include <cstdio>

using namespace mgpu;

struct idle_context_t : context_t {
  hipDeviceProp_t none = hipDeviceProp_t();
  int touched = 0;
  const hipDeviceProp_t& props() const override { return none; }
  int ptx_version() const override { return arch_version_gfx950; }
  hipStream_t stream() override { return touch(); }
  void* alloc(size_t, memory_space_t) override { return touch(); }
  void free(void*, memory_space_t) override { }
  void synchronize() override { }
  hipEvent_t event() override { return nullptr; }
  void timer_begin() override { }
  double timer_end() override { return 0; }
private:
  std::nullptr_t touch() {
    ++touched;
    throw cuda_exception_t(hipErrorNotSupported);
  }
};

static int failed = 0;

template<typename call_t>
static void refused(const char* what, call_t call) {
  idle_context_t context;
  hipError_t code = hipSuccess;
  try { call(context); } catch(const cuda_exception_t& e) { code = e.result; }
  if(hipErrorInvalidValue != code || context.touched) {
    printf("%s: code %d, %d calls of the context\n", what, (int)code,
      context.touched);
    failed = 1;
  }
}

template<typename call_t>
static void idle(const char* what, call_t call) {
  idle_context_t context;
  hipError_t code = hipSuccess;
  try { call(context); } catch(const cuda_exception_t& e) { code = e.result; }
  if(hipSuccess != code || context.touched) {
    printf("%s: code %d\n", what, (int)code);
    failed = 1;
  }
}

int main() {
  const int big = (1 << 30) + 1;
  float* x = nullptr;
  int* i = nullptr;
  auto lookup = [&](int count, int dim) {
    return [=](context_t& c) {
      embedding_lookup((const float*)x, 5, dim, (int64_t)0, i, count, 1.f, x,
        (int64_t)dim, c);
    };
  };
  refused("lookup of many", lookup(big, 1));
  refused("lookup of long rows", lookup(1, big));
  idle("lookup of none", lookup(0, big));

  auto grad = [&](int count, int num_rows, int dim) {
    return [=](context_t& c) {
      embedding_grad((const float*)x, (int64_t)0, i, count, num_rows, dim, 1.f,
        false, x, (int64_t)dim, c);
    };
  };
  refused("gradient of many", grad(big, 1, 1));
  refused("gradient of a long table", grad(1, big, 1));
  refused("gradient of long rows", grad(1, 1, big));
  idle("gradient of no rows", grad(5000, 0, big));
  idle("gradient of empty rows", grad(5000, 5, -1));

  auto loss = [&](int rows, int vocab, int top) {
    return [=](context_t& c) {
      distill_loss((const float*)x, (int64_t)0, rows, vocab, i,
        (const float*)x, top, 1.f, (const float*)x, x, x, c);
    };
  };
  auto dz = [&](int rows, int vocab, int top) {
    return [=](context_t& c) {
      distill_grad((const float*)x, (int64_t)0, rows, vocab, (const float*)x, i,
        (const float*)x, top, 1.f, (const float*)x, x, (int64_t)vocab, c);
    };
  };
  auto both = [&](int rows, int vocab, int top) {
    return [=](context_t& c) {
      distill_loss_and_grad((const float*)x, (int64_t)0, rows, vocab, i,
        (const float*)x, top, 1.f, (const float*)x, x, x, (int64_t)vocab, c);
    };
  };
  refused("loss, many entries", loss(1, 10, distill_max_top + 1));
  refused("gradient, many entries", dz(1, 10, distill_max_top + 1));
  refused("both, many entries", both(1, 10, distill_max_top + 1));
  refused("loss, long rows", loss(1, distill_max_vocab + 1, 1));
  refused("gradient, long rows", dz(1, distill_max_vocab + 1, 1));
  refused("both, long rows", both(1, distill_max_vocab + 1, 1));
  idle("loss of none", loss(0, 10, 1));

  auto draw = [&](int rows, int vocab) {
    return [=](context_t& c) {
      sample((const float*)x, (int64_t)0, rows, vocab, (const float*)x,
        (const float*)x, (const int*)i, (const float*)x, (const float*)x, 1.f,
        0, 1.f, 0.f, i, x, c);
    };
  };
  refused("draw from nothing", draw(1, 0));
  refused("draw from a negative number", draw(1, -5));
  refused("draw from too many", draw(1, sample_max_vocab + 1));
  idle("no draws", draw(0, 0));

  if(!failed) printf("rows limits: passed\n");
  return failed;
}
