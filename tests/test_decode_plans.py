"""The plans of the tree attention (csrc/tree_attention_plan.cuh), on the host: a call without a
workspace has no result to leave in one, and the workspace that is asked for holds every result of
either kernel. Compiled with nvcc into a small host program; no GPU."""

import subprocess

import pytest

from conftest import REPO

PROGRAM = r"""
#include <cstdio>
#include "tree_attention_plan.cuh"
using namespace ppyb200::tree;
int main() {
  for (long long capacity : {1, 60, 64, 128, 192, 256, 1000, 30000})
    for (long long nodes : {1, 2, 16, 17, 20, 40, 65, 130, 300})
      for (long long heads : {1, 2, 3, 8, 40})
        for (long long kv : {1, 2, 3, 8, 40})
          for (long long batch : {1, 2, 7})
            for (long long dim : {8, 32, 40, 64, 128})
              for (int wide = 0; wide < 2; ++wide) {
                Args a = {};
                a.batch = batch; a.nodes = nodes; a.heads = heads; a.kv_heads = kv;
                a.head_dim = dim; a.capacity = capacity; a.dtype = PPYB200_BF16;
                if (heads % kv != 0 || (wide && !wide_fits(a))) continue;
                const Plan p = plan_for(a, wide != 0, 148);
                const long long rows = (p.deal.item_rows + 7) / 8 * 8, padded = dim <= 64 ? 64 : 128;
                // the largest offset that a result, its top or an item's CTAs are written behind
                const long long results = p.deal.streams == 1
                    ? 2ll * p.deal.grid : p.deal.streams * (p.deal.grid + kv * batch * p.deal.items);
                const long long end = results * rows * (padded + 2) * 4 + kv * batch * p.deal.items * 8;
                printf("%d %d %d %lld %lld\n", p.deal.join ? 1 : 0, p.deal.grid, p.deal.streams,
                       (long long)p.workspace, end);
              }
  return 0;
}
"""


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    from ppy_b200 import toolchain

    if toolchain.nvcc() is None:
        pytest.skip("nvcc is not here")
    work = tmp_path_factory.mktemp("plans")
    source = work / "plans.cu"
    source.write_text(PROGRAM)
    program = work / "plans"
    done = subprocess.run([toolchain.nvcc(), *toolchain.GENCODE, "-std=c++17",
                           "--expt-relaxed-constexpr", f"-I{toolchain.CSRC}",
                           f"-I{REPO / 'include'}", "-o", str(program), str(source)],
                          capture_output=True, text=True, check=False)
    assert done.returncode == 0, done.stderr
    out = subprocess.run([str(program)], capture_output=True, text=True, check=True).stdout
    return [tuple(map(int, line.split())) for line in out.splitlines()]


def test_results_go_to_a_workspace_or_nowhere(plans):
    alone = [p for p in plans if not p[0]]
    assert len(plans) > 1000 and len(alone) > 20
    for join, grid, streams, workspace, end in plans:
        # one CTA and one stream: every item is one segment, written out where it is computed
        assert join == (grid > 1 or streams > 1)
        assert workspace == (end if join else 0)
