"""The example's text, which needs no GPU."""
import importlib.util
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_corpus(tmp_path):
    spec = importlib.util.spec_from_file_location("moe_train", os.path.join(ROOT, "examples", "moe_train.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    text = example.corpus()              # of the interpreter that runs this, wherever it is installed
    assert text.dtype == torch.int64 and 1 << 16 <= text.numel() <= 4 << 20 and 0 <= text.min() and text.max() < 256
    assert example.corpus(limit=1 << 17).numel() == 1 << 17
    (tmp_path / "a.py").write_bytes(b"x" * 70000)
    assert torch.equal(example.corpus(str(tmp_path)), torch.full((70000,), ord("x")))
    (tmp_path / "a.py").write_bytes(b"x" * 99)
    with pytest.raises(RuntimeError, match="99 bytes"):
        example.corpus(str(tmp_path))
