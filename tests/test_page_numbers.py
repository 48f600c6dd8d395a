"""What ``copy_pages`` takes for a page number (no GPU)."""
import pytest
import torch

import tiny_vllm_b200  # noqa: F401
from tiny_vllm_b200.attention import cuda as A


@pytest.mark.parametrize("src,dst", [([True], [0]), ([1], [False]), ([0, True], [3, 4])])
def test_truth_values_are_no_page_numbers(monkeypatch, src, dst):
    monkeypatch.setattr(A, "_require_cuda", lambda *tensors: None)
    with pytest.raises(ValueError, match="lists of page numbers"):
        A.copy_pages(torch.zeros(2, 5, 16, 2, 64, dtype=torch.bfloat16), src, dst)
