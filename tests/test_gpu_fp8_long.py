"""More rows than a grid of 2^32 threads holds, on a real MI355X (one column or two, so that memory stays small).

Assertions compare numbers: pytest's report of a failed one would take minutes over tensors of this size."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def need(dev, gib):
    if torch.cuda.mem_get_info(dev)[0] < gib << 30:
        pytest.skip("not enough free memory")


def test_choice_of_more_rows_than_a_grid_holds(dev):
    from src import ops
    need(dev, 8)
    T = 2 ** 26 + 2 ** 21 + 64
    z = torch.zeros(T, 2, device=dev, dtype=torch.bfloat16)
    u = torch.full((T,), 0.75, device=dev)
    u[5::7] = 0.25
    ids = torch.full((T,), 9, device=dev)
    ids[3::11] = 4
    got = ops.sample_tokens(z, u, ids=ids, mask_token_id=9)
    want = (u > 0.5).long()
    wrong = int((got != torch.where(ids == 9, want, ids)).sum())
    assert wrong == 0


@pytest.mark.parametrize("norm", [False, True])
def test_rows_of_more_blocks_than_a_grid_holds(dev, norm):
    from src import ops
    need(dev, 24)
    T = 2 ** 28 + 2 ** 27 + 21
    x = torch.ones(T, 1, device=dev, dtype=torch.bfloat16)
    x[1::3] = 0.5
    x[T - 1] = -2.0
    w = torch.full((1,), 3.0, device=dev)
    q, s = ops.rms_norm_fp8(x, w, 0.0)[:2] if norm else ops.quantize_fp8(x)
    q, s = q[:, 0].contiguous().view(torch.uint8), s[:, 0].view(torch.uint8)
    x = x[:, 0]
    # e4m3 256, 128 ..: of a power of two in [2^-8 448, 2 448) the value held is 256; 3 = 384 * 2^-7
    if norm:
        wrong = int((s != 127 - 7).sum()), int((q[:-1] != 0x7c).sum()), int(q[-1]) - 0xfc
    else:
        code = torch.full((T,), 119, dtype=torch.uint8, device=dev)
        code[x == 0.5] = 118
        code[T - 1] = 120
        wrong = int((s != code).sum()), int((q[:-1] != 0x78).sum()), int(q[-1]) - 0xf8
    assert wrong == (0, 0, 0)


@pytest.mark.parametrize("rd", [torch.bfloat16, torch.float32, None])
def test_launches_join_without_a_seam(dev, rd):
    """Rows around 2^23, where the norm's first launch ends, with strides of their own."""
    from src import ops
    need(dev, 16)
    T, d = 2 ** 23 + 9, 24
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn(T, 40, generator=g, device=dev, dtype=torch.bfloat16)[:, :d]
    r = None if rd is None else torch.randn(T, 32, generator=g, device=dev, dtype=rd)[:, :d]
    w = torch.rand(d, generator=g, device=dev) + 0.5
    q, s, st = ops.rms_norm_fp8(x, w, 1e-6, residual=r)
    at = slice(2 ** 23 - 9, None)
    q2, s2, st2 = ops.rms_norm_fp8(x[at], w, 1e-6, residual=None if r is None else r[at])
    first = ops.rms_norm_fp8(x[:9], w, 1e-6, residual=None if r is None else r[:9])
    same = [torch.equal(a.float(), b.float()) for a, b in ((q[at], q2), (s[at], s2), (st[at], st2), (q[:9], first[0]), (st[:9], first[2]))]
    assert same == [True] * 5
