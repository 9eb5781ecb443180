// host_arith.cu -- the library's host arithmetic, compiled on its own for tests
// that need no GPU (tests/test_operators_host.py).
#include "../355_1_trans_b200/csrc/host.cuh"
#include "../355_1_trans_b200/csrc/layer_norm.cuh"

#define TEST_API extern "C" __attribute__((visibility("default")))

// The plan of an MX GEMM on a device of `sms` SMs: out = {num_kb, split, kb_per}.
TEST_API void plan_mx(int m, int n, int k, int fp4, int kernel, int split_k, int sms, long long* out) {
  bsgemm_args a{};
  a.m = m;
  a.n = n;
  a.k = k;
  a.batch = 1;
  a.kernel = kernel;
  a.split_k = split_k;
  DevInfo dev;
  dev.sms = sms;
  MxPlan pl;
  mx_plan(a, fp4 != 0, dev, pl, true);
  out[0] = pl.num_kb;
  out[1] = pl.split;
  out[2] = pl.kb_per;
}

// The copies of the layer norm gradient's ring that are in flight when the wait for
// `row` at (stage, phase) has run out: out = {stage, parity} each; their number.
TEST_API int ring_pending(int row, int step, int rows, int stages, int stage, unsigned phase, int* out) {
  int n = 0, at;
  uint32_t parity;
  while (bsg::LnRing::pending(n, row, step, rows, stages, stage, phase, at, parity)) {
    out[2 * n] = at;
    out[2 * n + 1] = static_cast<int>(parity);
    ++n;
  }
  return n;
}
