"""Relation weights of 16-bit rows that start and end anywhere within 16 bytes, with histories up to the last column."""
import pytest
import torch

pytestmark = pytest.mark.gpu


# rows that stay in registers (256 and 512 threads), of every length within a piece of eight
@pytest.mark.parametrize("n", [4099 + 2 * i for i in range(4)] + [8188, 9411, 11763, 16371])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_last_columns_in_the_history(n, dt):
    from flashlog_b200 import attention
    rows, used = 320, 24
    g = torch.Generator().manual_seed(n)
    pitch = n + 8 - n % 8 + 1  # odd: a row starts at each of the eight places within 16 bytes
    z = (torch.randn(rows, pitch, generator=g) * 1.5).to(dt).cuda()[:, :n]
    history = torch.randint(0, n, (rows, used), generator=g)
    history[:, :8] = torch.arange(n - 8, n)
    history[::3, 8:16] = torch.arange(8)
    history[:, 20:] = n - 1
    history = history.cuda()
    w = attention.relation_weights(z, tau=0.8, history=history, repetition=1.3, frequency=0.2, presence=0.4)
    count = torch.zeros(rows, n, dtype=torch.float64, device=z.device)
    count.scatter_add_(1, history, torch.ones_like(history, dtype=torch.float64))
    u = z.double()
    u = torch.where(count > 0, torch.where(u > 0, u / 1.3, u * 1.3) - 0.2 * count - 0.4, u)
    want = torch.softmax(u / 0.8, 1)
    # an exponent's argument of at most 20 is off by a few roundings of 2^-24 of it, a sum of positive terms by fewer
    assert bool(((w - want).abs() <= 2.0 ** -16 * want + 1e-38).all())
    assert float((w.double().sum(1) - 1).abs().max()) <= 2.0 ** -16
