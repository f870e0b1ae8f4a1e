"""Operands that are packed but do not begin at a multiple of 16 bytes (a part of a larger buffer) give the same bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _shifted(x, by):
    buf = torch.empty(x.numel() + by, device="cuda", dtype=x.dtype)
    y = buf[by:].view(x.shape)
    y.copy_(x)
    assert y.is_contiguous() and y.data_ptr() % 16 != 0
    return y


@pytest.mark.parametrize("by", [1, 4])
@pytest.mark.parametrize("D", [64, 128, 160])
def test_packed_prompts(D, by):
    from acctransformer_b200 import flash_attention_packed
    q, k, v = (torch.randn(200, heads, D, device="cuda").half() for heads in (4, 2, 2))
    cu = torch.tensor([0, 130, 200], dtype=torch.int32, device="cuda")
    want = flash_attention_packed(q, k, v, cu)
    assert torch.equal(flash_attention_packed(_shifted(q, by), _shifted(k, by), _shifted(v, by), cu), want)


@pytest.mark.parametrize("by", [1, 4])
def test_cache(by):
    from acctransformer_b200 import Kv4Cache
    B, N_kv, D = 2, 2, 64
    lens, cu = torch.tensor([30, 9], dtype=torch.int32, device="cuda"), torch.tensor([0, 30, 39], dtype=torch.int32, device="cuda")
    k, v = (torch.randn(39, N_kv, D, device="cuda").half() for _ in range(2))
    q = torch.randn(B, 4, 1, D, device="cuda").half()
    one, two = (Kv4Cache(B, N_kv, 32, D) for _ in range(2))
    one.append(k, v, torch.zeros_like(lens), cu)
    two.append(_shifted(k, by), _shifted(v, by), torch.zeros_like(lens), cu)
    for x, y in zip(one.read(torch.zeros_like(lens), cu, total=39), two.read(torch.zeros_like(lens), cu, total=39)):
        assert torch.equal(x, y)
    assert torch.equal(one.decode(q, lens), two.decode(_shifted(q, by), lens))
