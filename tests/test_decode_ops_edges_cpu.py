"""What the decode step's operators do at their edges, as far as that can be seen without a GPU:
index arithmetic compiled for the host, and refusals."""

import os
import subprocess

import pytest
import torch

import newt_b200
from newt_b200 import ops
from newt_b200.runtime import abi
from test_decode_ops_cpu import P, _append, _attend, _cache, _grad, _rms, _score

CSRC = os.path.join(os.path.dirname(newt_b200.__file__), "csrc")

COLUMNS = r"""
#include <cstdio>
#include <vector>
#include "shifted_row.cuh"
using nb200::ShiftedRow;

#define CHECK(what) if (!(what)) { std::printf("n=%d m=%d E=%d shift=%d: %s\n", n, m, E, shift, #what); return 1; }

int check(int n, int m, int E, int shift, int threads) {
  const ShiftedRow row(n, m, E);
  const int groups = (n + (1 << shift) - 1) >> shift;
  std::vector<int> seen(n);
  CHECK(row.singles() >= 0 && row.singles() < 2 * E);
  for (int i = 0; i < row.singles(); ++i) {
    CHECK(row.single(i) >= 0 && row.single(i) < n);
    ++seen[row.single(i)];
  }
  for (int column = -m; column < n + threads * E; column += E) {
    const int before = row.group_before(column, shift), from = row.group_from(column, shift);
    CHECK(before >= -1 && before < groups && from >= -1 && from < groups);
    CHECK((before >= 0) == (m && row.whole(column)));       // nothing from a vector that is left out
    if (!row.whole(column)) continue;
    CHECK(column % E == (E - m) % E && column + E <= n);
    CHECK(m == 0 || column - row.head + 2 * E <= n);        // the weight's second vector
    for (int j = 0; j < E; ++j) {
      ++seen[column + j];
      CHECK(((column + j) >> shift) == (j < m ? before : from));
    }
  }
  for (int c = 0; c < n; ++c) CHECK(seen[c] == 1);
  return 0;
}

int main() {
  for (int E = 4; E <= 8; E += 4)
    for (int m = 0; m < E; ++m)
      for (int shift = 5; shift <= 7; ++shift)
        for (int n = 1; n <= 700; ++n)
          if (check(n, m, E, shift, 32)) return 1;
  return 0;
}
"""


def test_columns_of_shifted_rows_and_their_groups(tmp_path):
    """Every column of a row that starts off a vector boundary is taken once, and no group outside of the
    row's is touched."""
    source, program = tmp_path / "columns.cpp", tmp_path / "columns"
    source.write_text(COLUMNS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", CSRC, str(source), "-o", str(program)], check=True)
    done = subprocess.run([str(program)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout + done.stderr


def test_calls_that_would_lose_a_gradient_are_refused():
    x, w = torch.zeros(4, 64), torch.zeros(64)
    cache = ops.new_kv_cache(8, 2, 16, 64, device="cpu")
    kv = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    table = torch.zeros(2, 4, dtype=torch.int32)
    lengths, offsets = torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    q = torch.zeros(2, 1, 4, 64, dtype=torch.bfloat16)

    def wants(t):
        return t.clone().requires_grad_()

    calls = {"x": lambda: ops.rmsnorm(wants(x), w), "weight": lambda: ops.rmsnorm(x, torch.nn.Parameter(w)),
             "residual": lambda: ops.rmsnorm(x, w, residual=wants(x)), "out": lambda: ops.rmsnorm(x, w, out=wants(x)),
             "k": lambda: ops.kv_append(cache, wants(kv), kv, table, lengths, offsets, 1),
             "v": lambda: ops.kv_append(cache, kv, wants(kv), table, lengths, offsets, 1),
             "q": lambda: ops.kv_attention(wants(q), cache, table, lengths),
             "cache.v_scales": lambda: ops.kv_attention(
                 q, cache._replace(v_scales=wants(cache.v_scales)), table, lengths)}
    for name, call in calls.items():
        with pytest.raises(RuntimeError, match=f"'{name}' requires a gradient.*no backward"):
            call()
        with torch.no_grad(), pytest.raises(TypeError, match="must be a CUDA tensor"):   # the next check
            call()
        with torch.inference_mode(), pytest.raises(TypeError, match="must be a CUDA tensor"):
            call()


@pytest.mark.parametrize("call", [
    lambda: _rms(x=P + 1), lambda: _rms(w=P + 1), lambda: _rms(out=P + 1), lambda: _rms(res=P + 1),
    lambda: _rms(res=P, res_out=P + 1), lambda: _rms(x=P + 2, dtype=abi.F32, out_dtype=abi.F32),
    lambda: _rms(out_dtype=abi.E4M3, scales=P + 2), lambda: _append(_cache(ks=P + 2)),
    lambda: _append(k=P + 1), lambda: _append(v=P + 1), lambda: _append(table=P + 2),
    lambda: _append(starts=P + 1), lambda: _append(offsets=P + 2), lambda: _attend(_cache(vs=P + 1)),
    lambda: _attend(q=P + 1), lambda: _attend(out=P + 1), lambda: _attend(table=P + 2),
    lambda: _attend(lengths=P + 2), lambda: _score(logits=P + 2), lambda: _score(logits=P + 1, dtype=abi.F16),
    lambda: _score(tokens=P + 4), lambda: _score(logprob=P + 2), lambda: _score(top=2, best=P, index=P + 4),
    lambda: _score(top=2, best=P + 1, index=P), lambda: _grad(logits=P + 2), lambda: _grad(out=P + 3),
    lambda: _grad(tokens=P + 4), lambda: _grad(lse=P + 1), lambda: _grad(entropy=P + 2), lambda: _grad(g=P + 2),
    lambda: _grad(ge=P + 1, dtype=abi.BF16)])
def test_the_library_refuses_what_does_not_start_on_an_element(call):
    assert call() == abi.E_INVALID
    assert "multiple of" in abi.last_error()
