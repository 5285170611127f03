"""GPU: bucket_attention without gradients where the keys are split into runs: ragged lengths around the last bucket edge, where a
run's last tile holds only far keys but reaches past them."""
import pytest
import torch

from tests._transformer_ref import attention64, held, poison

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _inputs(B, Tq, Tk, H, Hk, D, dtype, nb=32, seed=0):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(B, T, h, D, generator=g) for T, h in ((Tq, H), (Tk, Hk), (Tk, Hk)))
    # biases that tell heads and buckets apart: what another head or bucket would leave is far off
    table = 0.37 * torch.arange(nb * H, dtype=torch.float32).view(nb, H) % 7 + 11.0 * torch.arange(H)
    return [t.to(dtype).to(DEV) for t in (q, k, v)] + [table.to(DEV)]


def _fill_lds(heads):
    """Runs that leave buckets and biases of their own in the compute units' LDS."""
    from asr_amd.Models.transformer_ops import bucket_attention
    q, k, v, t = _inputs(1, 256, 256, heads, heads, 64, torch.float32, seed=9)
    bucket_attention(q, k, v, 50.0 - t * 5)


def _check(q, k, v, table, *, lengths=None, offset=None, causal=False, reach=128):
    from asr_amd.Models.transformer_ops import bucket_attention
    _fill_lds(q.shape[2])
    poison()
    got = bucket_attention(q, k, v, table, lengths=lengths, offset=offset, causal=causal, max_distance=reach)
    wide = table if table is not None else torch.zeros(2 if causal else 4, q.shape[2], device=DEV)
    held(got, attention64(*(x.double() for x in (q, k, v, wide)), None, q.dtype, lengths=lengths, keep=None, offset=offset, causal=causal,
                          reach=reach, scale=q.shape[-1] ** -0.5, train=False)[0])


@pytest.mark.parametrize("causal", [False, True], ids=["both-sides", "causal"])
@pytest.mark.parametrize("length", [97, 101, 110, 127])
def test_one_utterance_with_ragged_keys(length, causal):
    q, k, v, t = _inputs(1, 374, 374, 4, 4, 64, torch.float32)
    n = torch.tensor([length], device=DEV, dtype=torch.int32)
    _check(q, k, v, t, lengths=n, causal=causal)
    _check(q, k, v, None, lengths=n, causal=causal)


@pytest.mark.parametrize("causal", [False, True], ids=["both-sides", "causal"])
def test_two_long_utterances(causal):
    q, k, v, t = _inputs(2, 1000, 1000, 1, 1, 32, torch.float32)
    for a in range(500, 1000, 83):
        _check(q, k, v, t, lengths=torch.tensor([a, a + 41], device=DEV, dtype=torch.int32), causal=causal)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("causal", [False, True], ids=["both-sides", "causal"])
def test_one_query_at_every_place_behind_a_short_cache(dtype, causal):
    """Queries from the last bucket's border to a tile beyond it behind the last key."""
    Tk, n, reach = 120, 101, 40
    offs = torch.arange(n - 1 + reach // 2, n + reach + 32, device=DEV, dtype=torch.int32)
    B = len(offs)
    q, k, v, t = _inputs(B, 1, Tk, 4, 2, 32, dtype, nb=16)
    _check(q, k, v, t, lengths=torch.full((B,), n, device=DEV, dtype=torch.int32), offset=offs, causal=causal, reach=reach)
    _check(q, k, v, None, lengths=torch.full((B,), n, device=DEV, dtype=torch.int32), offset=offs, causal=causal, reach=reach)


def test_every_remainder_of_a_tile():
    B, reach = 32, 64
    n = torch.arange(65, 65 + B, device=DEV, dtype=torch.int32)
    for more in (0, 1, 15, 30):
        q, k, v, t = _inputs(B, 1, 100, 8, 1, 64, torch.bfloat16, nb=16, seed=more)
        _check(q, k, v, t, lengths=n, offset=n - 1 + reach + more, causal=True, reach=reach)


@pytest.mark.parametrize("B,Tq,Tk,H,Hk,D,causal", [(3, 1, 700, 8, 2, 64, True), (1, 1, 3000, 4, 4, 128, True), (2, 5, 333, 6, 3, 40, False),
                                                   (1, 150, 374, 4, 4, 40, False), (2, 33, 1000, 2, 1, 128, True), (1, 100, 500, 2, 2, 96, False)])
def test_bfloat16_probabilities_keep_16_bits(B, Tq, Tk, H, Hk, D, causal):
    """Split keys: held to the tolerance of training's forward, whose probabilities have at least 16 bits."""
    from asr_amd.Models.transformer_ops import bucket_attention
    g = torch.Generator().manual_seed(11)
    q, k, v = (torch.randn(B, T, h, D, generator=g).to(torch.bfloat16).to(DEV) for T, h in ((Tq, H), (Tk, Hk), (Tk, Hk)))
    t = torch.randn(32, H, generator=g).to(DEV)
    off = torch.full((B,), Tk - Tq, device=DEV, dtype=torch.int32)
    got = bucket_attention(q, k, v, t, offset=off, causal=causal)
    held(got, attention64(*(x.double() for x in (q, k, v, t)), None, torch.bfloat16, lengths=None, keep=None, offset=off, causal=causal,
                          reach=128, scale=D ** -0.5, train=True)[0])
