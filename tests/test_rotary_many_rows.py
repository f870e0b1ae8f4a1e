"""Rotary positions where a call has more threads than 32 bits count: plans whose half is odd, or twice an odd number, have small units."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sections,adjacent,N,rows", [((1,), False, 1, 33_900_000), ((2,), False, 1, 68_300_000), ((3,), True, 1, 68_000_000), ((1,), False, 5, 17_000_000)],
                         ids=["1", "2", "adjacent", "heads"])
def test_all_rows_are_turned(sections, adjacent, N, rows):
    from acctransformer_b200 import Rotary
    D = 128
    # units of the row's values, threads of four heads each
    vec = 2 if adjacent else sections[0]
    turned = 2 * sections[0] if adjacent else sections[0]
    units = (turned + D - 2 * sections[0]) // vec
    assert rows * units * ((N + 3) // 4) > 2 ** 32
    assert torch.cuda.mem_get_info()[0] > 5 * rows * N * D
    rotary = Rotary(D, sections, adjacent=adjacent)
    x = torch.empty(rows, N, D, dtype=torch.float16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(1))
    pos = torch.randint(0, 1000, (rows,), dtype=torch.int32, device="cuda")
    y = rotary(x, None, pos)[0]
    for at in range(0, rows, 1 << 20):      # (a row's values do not depend on how many there are: calls of few threads)
        part = slice(at, min(rows, at + (1 << 20)))
        assert torch.equal(y[part], rotary(x[part], None, pos[part])[0])


@pytest.mark.parametrize("B,S,wide,shared", [(3, 23_000_001, False, False), (5, 7_000_003, True, False), (2, 34_000_000, True, True), (34_000, 1000, False, True)])
def test_batches(B, S, wide, shared):
    """[B, 1, S, D], a launch each of some batch entries, or of a part of one."""
    from acctransformer_b200 import Rotary
    D, T = 128, B * S
    assert T * 127 > 2 ** 32
    rotary = Rotary(D, (1,), base=100.0)
    x = torch.empty(B, 1, S, D, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(1))
    pos = torch.randint(0, 1000, (S,) if shared else (B, S), dtype=torch.int64 if wide else torch.int32, device="cuda")
    y = rotary(x, None, pos)[0].view(T, D)
    rows, at = x.view(T, 1, D), pos.expand(B, S).reshape(T)
    for i in range(0, T, 1 << 20):
        part = slice(i, min(T, i + (1 << 20)))
        assert torch.equal(y[part], rotary(rows[part], None, at[part])[0].view(-1, D))
