"""Window decode at the ends of the rule that cuts rows into parts: 31 pages (whole), 32 and more (four parts), few rows."""

import pytest
import torch

from femtovllm import workloads
from helpers import assert_close
from test_window_gpu import free_hidden_blocks, run_decode

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window,sinks", [(491, 5), (492, 5), (507, 5), (512, 0), (520, 3)])
@pytest.mark.parametrize("lens", [[30000], [700, 496], [512, 513, 1, 16]])
def test_rows_of_32_pages(ops, gpu, lens, window, sinks, dtype):
    w = workloads.make_paged_workload("parts", [(L - 1, 1) for L in lens], 8, 2, dtype=dtype, seed=len(lens) + window)
    free_hidden_blocks(w, window, sinks)
    out, want = run_decode(ops, w, gpu, window, sinks)
    assert_close(out, want, dtype, f"window {window} lens {lens}")
    again, _ = run_decode(ops, w, gpu, window, sinks)
    assert torch.equal(again, out)
