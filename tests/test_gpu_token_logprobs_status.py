"""The status word of the log probabilities: one int32, which the kernel sets bits of as a word."""
import pytest
import torch

from socket_b200 import _lib, few_rows

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("library", ["step", "blocks"])
@pytest.mark.parametrize("dtype,n", [(torch.uint8, 1), (torch.int8, 4), (torch.bool, 1), (torch.int16, 2), (torch.int64, 1), (torch.float32, 1),
                                     (torch.int32, 0), (torch.int32, 2)])
def test_status_words_that_are_refused(dtype, n, library):
    x, tokens = torch.randn(4, 100, device=DEV), torch.tensor([1, 2, 3, 4], device=DEV)          # nothing to flag
    with pytest.raises(AssertionError):
        few_rows.token_logprobs(x, tokens, status=torch.zeros(n, dtype=dtype, device=DEV), library=library)


@pytest.mark.parametrize("library", ["step", "blocks"])
@pytest.mark.parametrize("shape", [(), (1,), (1, 1)])
def test_status_words_that_are_taken(shape, library):
    x, flag = torch.randn(4, 100, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)
    word = flag[1].view(shape)                                # beside words of others
    few_rows.token_logprobs(x, torch.tensor([1, 2, 3, 4], device=DEV), status=word, library=library)
    assert flag.tolist() == [0, 0, 0]
    few_rows.token_logprobs(x, torch.tensor([1, 2, -1, 4], device=DEV), status=word, library=library)
    assert flag.tolist() == [0, _lib.SK_DEV_INDEX_OUT_OF_RANGE, 0]
