"""More rows of classes, or sequences, than one launch has workgroups for, on the GPU: each of them still gets its results."""
import pytest
import torch

from gpu_util import call

pytestmark = pytest.mark.gpu


def _rows(rows, n, dtype):
    """Rows of dyadic numbers that tell them apart; cheap to make."""
    r = torch.arange(rows, device="cuda", dtype=torch.int32)
    x = torch.empty(rows, n, dtype=dtype, device="cuda")
    for j in range(n):
        x[:, j] = ((r * (2 * j + 3) + j * 7) % 61).to(torch.float32) * 0.125
    return x


@pytest.mark.parametrize("k", [2, 257])
def test_top_k_of_many_rows(k):
    # k above 256 takes 256 threads a row: 2^24 rows are 2^32 of them
    n, rows = 3, 2 ** 25 + 5 if k == 2 else 2 ** 24 + 5
    print("many rows: top_k", k, flush=True)
    x = _rows(rows, n, torch.bfloat16)
    value = torch.full((rows, k), 77.0, device="cuda")
    index = torch.full((rows, k), 77, dtype=torch.int32, device="cuda")
    norm = torch.full((rows,), 77.0, device="cuda")
    call("anode_gpu_top_k_rows_bf16", n, rows, 0, k, 1.0, x, value, index, norm)
    want, place = torch.sort(x.float(), dim=1, descending=True, stable=True)
    some = min(n, k)
    assert bool((value[:, :some] == want[:, :some]).all()) and bool((index[:, :some] == place[:, :some]).all())
    assert bool((value[:, some:] == -float("inf")).all()) and bool((index[:, some:] == -1).all())
    # three terms: the log-sum-exp of values to 8 is off by some half steps of a number to 9.1 (2^-21 each)
    assert float((norm.double() - torch.logsumexp(x.double(), 1)).abs().max()) <= 8 * 2.0 ** -21


def test_distill_of_many_rows():
    n, rows = 3, 2 ** 25 + 5
    print("many rows: distill", flush=True)
    x = _rows(rows, n, torch.float32)
    label = (torch.arange(rows, device="cuda", dtype=torch.int32) % n)
    value, dy = torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda")
    want = torch.logsumexp(x.double(), 1) - x.double().gather(1, label.long()[:, None])[:, 0]
    dx_want = torch.softmax(x.double(), 1)
    dx_want.scatter_add_(1, label.long()[:, None], torch.full((rows, 1), -1.0, dtype=torch.float64, device="cuda"))
    for fused in (True, False):
        loss, top, total = (torch.full((rows,), 77.0, device="cuda") for _ in range(3))
        dx = torch.full_like(x, 77.0)
        if fused:
            call("anode_gpu_softmax_distill_fused_fwd_bwd_rows_f32", n, rows, 0, 1, 1.0, x, value, label, None, dy, loss, top, total, dx)
        else:
            call("anode_gpu_softmax_distill_rows_f32", n, rows, 0, 1, 1.0, x, value, label, None, loss, top, total)
            call("anode_gpu_softmax_distill_bwd_rows_f32", n, rows, 0, 1, 1.0, dy, x, value, label, None, top, total, dx)
        assert bool((top == x.amax(1)).all())
        assert float((loss.double() - want).abs().max()) <= 16 * 2.0 ** -21
        assert float((dx.double() - dx_want).abs().max()) <= 32 * 2.0 ** -24


@pytest.mark.parametrize("drafted", [0, 1])
def test_verify_many_sequences_of_few_classes(drafted):
    n, B = 3, 2 ** 24 + 5
    print("many sequences", drafted, flush=True)
    r = torch.arange(B, device="cuda", dtype=torch.int32)
    target = torch.empty(B, drafted + 1, n, device="cuda")
    for i in range(drafted + 1):                       # dyadic weights that sum to one
        a = ((r + i) % 3).float() * 0.25
        target[:, i, 0], target[:, i, 1], target[:, i, 2] = a, 0.25, 0.75 - a
    draft = torch.full((B, drafted, n), 0.25, device="cuda")
    token_in = (r % 4).view(B, 1)[:, :drafted].contiguous()      # a class outside now and then
    accept = ((r % 5).float() * 0.25).view(B, 1)[:, :drafted].contiguous()
    pick = ((r % 7).float() * 0.125).contiguous()
    token = torch.full((B, drafted + 1), 77, dtype=torch.int32, device="cuda")
    accepted = torch.full((B,), 77, dtype=torch.int32, device="cuda")
    some = torch.zeros(1, device="cuda")
    call("anode_gpu_verify_draft_packed_f32", n, drafted, B, target, draft if drafted else some,
         token_in if drafted else some.int(), None, accept if drafted else some, pick, token, accepted)
    taken = torch.zeros(B, dtype=torch.bool, device="cuda")
    if drafted:
        t = token_in[:, 0].long()
        p = target[:, 0].gather(1, t.clamp(max=2)[:, None])[:, 0]
        taken = (t < 3) & (accept[:, 0] * 0.25 < p)
    row = (torch.where(taken[:, None], target[:, -1], target[:, 0]) if drafted else target[:, 0]).double()
    if drafted:
        rest = (row - 0.25).clamp(min=0.0)
        row = torch.where((~taken & (rest.sum(1) > 0))[:, None], rest, row)
    border = pick.double() * row.sum(1)                # (every sum is exact)
    over = [(row[:, 0] > border) & (row[:, 0] > 0), (row[:, 0] + row[:, 1] > border) & (row[:, 1] > 0)]
    drawn = torch.where(over[0], 0, torch.where(over[1], 1, 2)).int()
    assert bool((accepted == taken.int()).all())
    if drafted:
        assert bool((token[:, 0] == torch.where(taken, token_in[:, 0], drawn)).all())
        assert bool((token[:, 1] == torch.where(taken, drawn, -1)).all())
    else:
        assert bool((token[:, 0] == drawn).all())
