"""Rows that the log probabilities' 31-bit counts cannot hold are refused before anything is launched (CPU: the
addresses are never used)."""

import pytest

torch = pytest.importorskip("torch")

INVALID, OUT_OF_RANGE = 16, 17
F32, BF16, F16 = 0, 1, 2


def call(pkg, vocab, dtype, top_k=0, rows=1):
    at = 1 << 20  # (any aligned address)
    args = pkg.serving._LOGPROBS.pack(at, 0, 0, at, at, at, 1 << 40, dtype, rows, vocab, top_k)
    return pkg.load_library().tl_token_logprobs(args, None)


@pytest.mark.parametrize("dtype,size", [(F32, 4), (BF16, 2), (F16, 2)])
@pytest.mark.parametrize("over", ["limit", "2^31 bytes", "int32"])
def test_long_rows_are_refused(pkg, dtype, size, over):
    if torch.cuda.is_available():
        pytest.skip("the addresses are not a GPU's")
    vocab = {"limit": (2 ** 31 - 2 ** 17) // size, "2^31 bytes": 2 ** 31 // size, "int32": 2 ** 31 - 1}[over]
    for top_k in (0, 5):
        assert call(pkg, vocab, dtype, top_k) == OUT_OF_RANGE
        assert call(pkg, vocab, dtype, top_k, rows=300) == OUT_OF_RANGE
    assert call(pkg, -vocab, dtype) == INVALID
