// embed.hip's kernels on the CPU.  Each tensor and the scratch end where a page begins that
// nothing may touch, or begin where one ends, and inputs can only be read: an access out
// of range ends the process.  The scratch begins as garbage, the outputs as NaN.
//   embed_on_cpu op n vocab embd bf16 norm accumulate kind front
// op: embed, vjp.  kind: uniform (some ids out of range), few, one, short (the first input
// with rows lacks one, which has to be noticed).  front: buffers begin at a page, not end at
// one.
#include <math.h>
#include <signal.h>
#include <unistd.h>

#include <random>
#include <string>

#include "hip/hip_runtime.h"

extern "C" __bf16 __truncsfbf2(float x) {
  uint32_t b = __builtin_bit_cast(uint32_t, x);
  b = (b & 0x7fffffffu) > 0x7f800000u ? b | 0x400000u : b + 0x7fffu + ((b >> 16) & 1);
  return __builtin_bit_cast(__bf16, (uint16_t)(b >> 16));
}

#include "embed.hip"

static bool front = false;
static char* guarded(size_t bytes, size_t align) {
  const size_t page = 4096, body = (bytes + page - 1) / page * page;
  char* p = (char*)mmap(nullptr, body + 2 * page, PROT_NONE, MAP_PRIVATE | MAP_ANONYMOUS | MAP_NORESERVE, -1, 0);
  if (p == MAP_FAILED || mprotect(p + page, body, PROT_READ | PROT_WRITE) != 0) abort();
  return p + page + (front ? 0 : (body - bytes) / align * align);
}
static void only_read(char* p, size_t bytes) {
  const uintptr_t page = 4096, a = (uintptr_t)p / page * page;
  if (mprotect((void*)a, ((uintptr_t)p + bytes - a + page - 1) / page * page, PROT_READ) != 0) abort();
}

namespace bdh {
bdh_status fail(bdh_status st, const std::string& msg) {
  fprintf(stderr, "%s\n", msg.c_str());
  return st;
}
bdh_status hip_fail(hipError_t, const char* what) { return fail(BDH_EHIP, what); }
bdh_status scratch(hipStream_t, int, size_t bytes, void** out, bool) {
  char* p = guarded(bytes, 4);
  memset(p, 0xa5, bytes);  // (ids and places far out of range)
  *out = p;
  return BDH_OK;
}
}  // namespace bdh

static void out_of_range(int, siginfo_t* info, void*) {
  fprintf(stderr, "access out of range at %p: workgroup %u %u, thread %u\n", info->si_addr, blockIdx.x, blockIdx.y,
          threadIdx.x);
  _exit(5);
}

int main(int argc, char** argv) {
  if (argc != 10) return 2;
  static char stack[65536];
  stack_t alt{stack, 0, sizeof(stack)};
  struct sigaction act{};
  act.sa_sigaction = out_of_range;
  act.sa_flags = SA_SIGINFO | SA_ONSTACK;
  if (sigaltstack(&alt, nullptr) != 0 || sigaction(SIGSEGV, &act, nullptr) != 0) return 2;
  const bool vjp = std::string(argv[1]) == "vjp", bf16 = atoi(argv[5]), norm = atoi(argv[6]), add = atoi(argv[7]);
  const int64_t n = atoll(argv[2]), V = atoll(argv[3]), D = atoll(argv[4]);
  const std::string kind = argv[8];
  front = atoi(argv[9]);
  const size_t size = bf16 ? 2 : 4;
  std::mt19937_64 rng((uint64_t)(n * 7 + V * 3 + D));
  std::normal_distribution<float> normal;
  const auto put = [&](char* p, int64_t i, float x) {
    if (bf16) ((__bf16*)p)[i] = (__bf16)x;
    else ((float*)p)[i] = x;
  };
  const auto get = [&](const char* p, int64_t i) { return bf16 ? (double)(float)((const __bf16*)p)[i] : ((const float*)p)[i]; };
  const auto tensor = [&](int64_t count, bool numbers) {
    char* p = guarded((size_t)count * size, size);
    for (int64_t i = 0; i < count; ++i) put(p, i, numbers ? 0.5f + normal(rng) : NAN);
    return p;
  };
  int32_t* tokens = (int32_t*)guarded((size_t)n * 4, 4);
  for (int64_t i = 0; i < n; ++i) {
    const int64_t u = (int64_t)(rng() % (uint64_t)(V + 4)) - 2;
    tokens[i] = (int32_t)(kind == "one" ? V / 2 : kind == "few" ? (rng() % 8 ? V / 3 + (int64_t)(rng() % 3) % V : u) : u);
  }
  char *table = tensor((kind == "short" && !vjp ? V - 1 : V) * D, true), *grad = vjp ? tensor((kind == "short" ? n - 1 : n) * D, true) : nullptr, *out = tensor(vjp ? V * D : n * D, add);
  std::vector<double> old((size_t)(vjp && add ? V * D : 0));
  for (size_t i = 0; i < old.size(); ++i) old[i] = get(out, (int64_t)i);
  only_read((char*)tokens, (size_t)n * 4);
  if (kind != "short") only_read(table, (size_t)(V * D) * size);
  if (vjp && kind != "short") only_read(grad, (size_t)(n * D) * size);
  bdh::EmbedArgs a{};
  a.tokens = tokens;
  a.n = n;
  a.vocab = V;
  a.embd = D;
  a.table = table;
  a.bf16 = bf16;
  a.norm = norm;
  a.scale = 1.5f;
  a.out = out;
  a.grad = grad;
  a.accumulate = add;
  uint64_t launches = 0;
  if ((vjp ? bdh::embed_tokens_vjp(a, nullptr, &launches) : bdh::embed_tokens(a, nullptr)) != BDH_OK) return 3;

  // The formula in 64 bits.  (That nothing is lost or counted twice: a relative share of the sums' sizes.)
  const double share = bf16 ? 1.0 / 128 : 1e-4;
  double worst = 0.0;
  const auto hold = [&](double got, double want, double magnitude) {
    const double off = fabs(got - want) / (share * (magnitude + 1e-3));
    if (!(off <= worst)) worst = off;
  };
  std::vector<double> s((size_t)D), e((size_t)D), m((size_t)D);
  const auto row = [&](int64_t v) {  // e: the table's row, or its norm; returns 1 / sigma
    double mean = 0, var = 0;
    for (int64_t c = 0; c < D; ++c) mean += e[(size_t)c] = get(table, v * D + c);
    if (!norm) return 1.0;
    mean /= (double)D;
    for (int64_t c = 0; c < D; ++c) var += (e[(size_t)c] -= mean) * e[(size_t)c];
    const double r = 1.0 / sqrt(var / (double)D + 1e-5);
    for (int64_t c = 0; c < D; ++c) e[(size_t)c] *= r;
    return r;
  };
  if (!vjp) {
    for (int64_t i = 0; i < n; ++i) {
      const bool there = tokens[i] >= 0 && tokens[i] < V;
      if (there) row(tokens[i]);
      for (int64_t c = 0; c < D; ++c) hold(get(out, i * D + c), there ? 1.5 * e[(size_t)c] : 0.0, there ? 4.0 : 0.0);
    }
  } else {
    std::vector<std::vector<int64_t>> of((size_t)V);
    for (int64_t i = 0; i < n; ++i)
      if (tokens[i] >= 0 && tokens[i] < V) of[(size_t)tokens[i]].push_back(i);
    for (int64_t v = 0; v < V; ++v) {
      std::fill(s.begin(), s.end(), 0.0);
      std::fill(m.begin(), m.end(), 0.0);
      for (const int64_t i : of[(size_t)v])
        for (int64_t c = 0; c < D; ++c) {
          s[(size_t)c] += 1.5 * get(grad, i * D + c);
          m[(size_t)c] += 1.5 * fabs(get(grad, i * D + c));
        }
      double most = 0;
      for (const double x : m) most = x > most ? x : most;
      if (norm && !of[(size_t)v].empty()) {
        const double r = row(v);
        double mean = 0, along = 0;
        for (int64_t c = 0; c < D; ++c) {
          mean += s[(size_t)c] / (double)D;
          along += s[(size_t)c] * e[(size_t)c] / (double)D;
        }
        for (int64_t c = 0; c < D; ++c) s[(size_t)c] = r * (s[(size_t)c] - mean - e[(size_t)c] * along);
        most *= 4 * r;
      }
      for (int64_t c = 0; c < D; ++c) {
        const double was = add ? old[(size_t)(v * D + c)] : 0.0;
        if (of[(size_t)v].empty()) {  // zeros, or as it was
          if (get(out, v * D + c) != was) worst = INFINITY;
        } else {
          hold(get(out, v * D + c), s[(size_t)c] + was, most + fabs(was));
        }
      }
    }
  }
  printf("worst %.3g\n", worst);
  return worst <= 1.0 ? 0 : 4;
}
