"""The lookup's gradient of a table past 256 GiB, which one launch of 64 bytes a thread cannot clear."""
import pytest

from helpers import twd

pytestmark = pytest.mark.gpu


def test_table_past_256_gib():
    import torch
    t = twd()
    vocab, d = (1 << 17) + 1, 1 << 20
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 2 * vocab * d + (6 << 30):
        pytest.skip("the table does not fit beside what else is on the device")
    table = torch.ones(vocab, d, dtype=torch.bfloat16, device="cuda:0")
    rows = torch.full((2, d), 3.0, device="cuda:0")
    grad = t.EmbedGrad(2, d)
    grad.run(rows, torch.tensor([vocab - 1, -1], dtype=torch.int32, device="cuda:0"), table)
    assert bool((table[vocab - 1] == 3).all())
    assert not any(bool(table[r:r + 512].any()) for r in range(0, vocab - 1, 512))
    grad.close()
    del table
    torch.cuda.empty_cache()
