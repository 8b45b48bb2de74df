"""embed_tokens and its gradient against the formulas in 64 bits, at the sizes where they can go wrong."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24                                              # half a step of float32 at one
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}     # half a step below the smallest normal number


def _reference(tokens, table, scale, encode, grad=None):
    """(z, its tolerance) or (dtable, its tolerance), in float64 on the CPU."""
    tok, tab = tokens.cpu().long().reshape(-1), table.double().cpu()
    v = scale * tab
    # roundings: the product, the difference (each moves exp by its size), exp and what it is given (2 steps)
    z = torch.exp(1.0 - v) if encode else v
    tol_z = (U * (v.abs() + (1.0 - v).abs() + 4.0) if encode else U * torch.ones_like(v)) * z.abs() * 1.01
    if grad is None:
        return z[tok], tol_z[tok]
    g = grad.double().cpu().reshape(-1, tab.shape[1])
    known = (tok >= 0) & (tok < tab.shape[0])
    tok, g = tok[known], g[known]
    s = torch.zeros_like(tab).index_add_(0, tok, g)
    size = torch.zeros_like(tab).index_add_(0, tok, g.abs())
    count = torch.zeros(tab.shape[0], dtype=torch.float64).index_add_(0, tok, torch.ones(len(tok), dtype=torch.float64))
    k = -scale * z if encode else torch.full_like(z, scale)
    # a sum of c terms in any order: at most c - 1 roundings of partial sums below `size`; then the factor's, and two products
    tol = 1.01 * k.abs() * size * (U * (count[:, None] + 2.0) + tol_z / z.abs().clamp(min=1e-30)) + HALF[table.dtype] * (k * s).abs() * 1.01
    return k * s, tol + TINY[table.dtype]


def _close(got, want, tol, what):
    bad = (got.double().cpu() - want).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}"


def _case(N, V, D, dtype, seed=0, zipf=True, bits=torch.int64):
    gen = torch.Generator().manual_seed(seed + N + V + D)
    u = torch.rand(N, generator=gen)
    tok = (torch.exp(u * torch.log(torch.tensor(V + 1.0))) - 1).long().clamp(0, V - 1) if zipf else (u * V).long().clamp(0, V - 1)
    tok = torch.randperm(V, generator=gen)[tok].to(bits)
    table = torch.rand(V, D, generator=gen).to(dtype)
    return tok.to(DEV), table.to(DEV), torch.randn(N, D, generator=gen).to(DEV)


@pytest.mark.parametrize("bits", [torch.int32, torch.int64])
@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("N,V,D", [(1, 1, 1), (7, 3, 5), (64, 1000, 64), (300, 40, 257), (1025, 2000, 100), (4100, 97, 36), (63, 2, 70), (128, 9, 300),
                                   (129, 9, 300), (100, 30000, 12), (256, 3, 40), (257, 3, 40)])
def test_forward_and_gradient(N, V, D, dtype, bits):
    import snntc_amd as snn
    tok, table, grad = _case(N, V, D, dtype, bits=bits)
    for scale, encode in [(1.0, True), (0.75, False), (-1.5, True)]:
        _close(snn.embed_tokens(tok, table, scale, encode), *_reference(tok, table, scale, encode), "z")
        d = snn.embed_tokens_grad(grad, tok, table, scale, encode)
        assert d.dtype == dtype and d.shape == table.shape
        _close(d, *_reference(tok, table, scale, encode, grad), "dtable")


@pytest.mark.parametrize("N,V,D,dtype", [(20000, 30, 64, torch.float32), (17000, 50000, 33, torch.bfloat16), (40000, 1, 20, torch.float32),
                                         (70001, 300000, 8, torch.float16), (33000, 5000, 300, torch.float32),
                                         (12288, 700, 12, torch.float32), (12289, 1023, 12, torch.float32), (16385, 1024, 7, torch.float32),
                                         (20000, 1200000, 4, torch.bfloat16), (600000, 77, 3, torch.float32)])
def test_many_tokens(N, V, D, dtype):
    """More positions than the short sort takes; tokens that occur tens of thousands of times; tables most of whose rows are unused."""
    import snntc_amd as snn
    tok, table, grad = _case(N, V, D, dtype)
    _close(snn.embed_tokens_grad(grad, tok, table, 0.5, True), *_reference(tok, table, 0.5, True, grad), "dtable")


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("N,D", [(67111, 1000), (16411, 4100), (67111, 1001)])
def test_outputs_larger_than_the_caches(N, D, dtype):
    """Rows do not know how many there are: the quarters of an output of more than 256 MB, by themselves."""
    import snntc_amd as snn
    tok, table, _ = _case(N, 300, D, dtype)
    tok[5] = -1
    z = snn.embed_tokens(tok, table, 0.5, True)
    for part in (slice(k * N // 4, (k + 1) * N // 4) for k in range(4)):
        assert torch.equal(z[part].nan_to_num(-1.0), snn.embed_tokens(tok[part], table, 0.5, True).nan_to_num(-1.0))


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("D", [1100, 1101])
def test_gradients_larger_than_the_caches(D, dtype):
    """Of more than 256 MB with the times: the same sums as of the columns by themselves, which are less."""
    import snntc_amd as snn
    N = 31007
    tok, table, grad = _case(N, 700, D, dtype)
    d = snn.embed_tokens_grad(grad, tok, table, 0.5, True)
    for part in (slice(0, 512), slice(512, D)):
        half = snn.embed_tokens_grad(grad[:, part], tok, table[:, part], 0.5, True)
        # the same terms in chunks of another length: each side is off by its own roundings
        _close(d[:, part], half.double().cpu(), 2 * _reference(tok, table[:, part], 0.5, True, grad[:, part])[1], "dtable")


def test_more_elements_than_32_bits_count():
    import snntc_amd as snn
    N, D = 2300007, 1000
    tok = torch.arange(N - 1, -1, -1, device=DEV)
    table = torch.rand(N, D, device=DEV).to(torch.bfloat16)
    z = snn.embed_tokens(tok, table, 0.5)
    assert torch.equal(z[-3:], 0.5 * table[:3].float().flip(0)) and torch.equal(z[:3], 0.5 * table[-3:].float().flip(0))
    d = snn.embed_tokens_grad(z, tok, table, 0.5)
    for k in range(0, N, 100000):                               # (halves and quarters of bfloat16 are exact)
        assert torch.equal(d[k:k + 100000], 0.25 * table[k:k + 100000])


def test_one_token_throughout_and_all_different():
    import snntc_amd as snn
    for tok in (torch.full((5000,), 6), torch.arange(5000), torch.arange(5000).flip(0), torch.arange(5000) // 64, torch.arange(5000) % 2):
        gen = torch.Generator().manual_seed(3)
        table, grad = torch.rand(5000, 40, generator=gen).to(DEV), torch.randn(5000, 40, generator=gen).to(DEV)
        _close(snn.embed_tokens_grad(grad, tok.to(DEV), table), *_reference(tok, table, 1.0, False, grad), "dtable")


def test_the_same_sums_on_every_call():
    import snntc_amd as snn
    for N in (3000, 50000):
        tok, table, grad = _case(N, 2000, 65, torch.float32)
        first = snn.embed_tokens_grad(grad, tok, table)
        assert all(torch.equal(first, snn.embed_tokens_grad(grad, tok, table)) for _ in range(3))


@pytest.mark.parametrize("N", [50, 30000])
def test_tokens_outside_the_table(N):
    import snntc_amd as snn
    tok, table, grad = _case(N, 100, 12, torch.float32)
    tok[::7] = -1
    tok[3::11] = 100
    tok[5::13] = 2 ** 40
    tok[6::13] = -2 ** 33                                    # (its low 32 bits are 0)
    out = (tok < 0) | (tok >= 100)
    z = snn.embed_tokens(tok, table, 1.0, True)
    assert torch.isnan(z[out]).all() and not torch.isnan(z[~out]).any()
    grad[out] = float("nan")
    _close(snn.embed_tokens_grad(grad, tok, table, 1.0, True), *_reference(tok, table, 1.0, True, grad), "dtable")


def test_shapes_strides_and_empty_inputs():
    import snntc_amd as snn
    tok, table, _ = _case(24, 50, 6, torch.float32)
    t3 = tok.view(2, 3, 4)
    assert torch.equal(snn.embed_tokens(t3, table), snn.embed_tokens(tok, table).view(2, 3, 4, 6))
    assert torch.equal(snn.embed_tokens(t3.permute(2, 0, 1), table), snn.embed_tokens(t3, table).permute(2, 0, 1, 3))
    wide = torch.rand(50, 13, device=DEV)
    assert torch.equal(snn.embed_tokens(tok, wide[:, 1:13:2]), snn.embed_tokens(tok, wide[:, 1:13:2].contiguous()))
    none = torch.zeros(0, dtype=torch.int64, device=DEV)
    assert snn.embed_tokens(none, table).shape == (0, 6)
    assert torch.equal(snn.embed_tokens_grad(torch.zeros(0, 6, device=DEV), none, table), torch.zeros_like(table))
    assert snn.embed_tokens(tok, table[:, :0]).shape == (24, 0)
    odd = torch.rand(50 * 6 + 1, device=DEV)[1:].view(50, 6)                  # 4-byte aligned rows only
    assert torch.equal(snn.embed_tokens(tok, odd), snn.embed_tokens(tok, odd.clone()))
    og = torch.randn(24 * 6 + 1, device=DEV)[1:].view(24, 6)
    assert torch.equal(snn.embed_tokens_grad(og, tok, odd), snn.embed_tokens_grad(og.clone(), tok, odd.clone()))


def test_refusals():
    import snntc_amd as snn
    tok, table, grad = _case(8, 5, 4, torch.float32)
    with pytest.raises(TypeError, match="int64 or int32"):
        snn.embed_tokens(tok.float(), table)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        snn.embed_tokens(tok, table.double())
    with pytest.raises(ValueError, match="2 dimensions"):
        snn.embed_tokens(tok, table[0])
    with pytest.raises(ValueError, match="empty table"):
        snn.embed_tokens(tok, table[:0])
    with pytest.raises(ValueError, match="grad must have shape"):
        snn.embed_tokens_grad(grad[:7], tok, table)
    with pytest.raises(TypeError, match="grad must be float32"):
        snn.embed_tokens_grad(grad.half(), tok, table)
    with pytest.raises(snn.SnntcLibraryError):
        snn.embed_tokens(tok.cpu(), table)


def test_layer_gradient_by_differences_and_streams():
    import snntc_amd as snn
    gen = torch.Generator().manual_seed(0)
    layer = snn.SNN_embedding(9, 3, scale=0.8, weight=torch.rand(9, 3, generator=gen).numpy()).to(DEV)
    tok = torch.tensor([[1, 1, 4], [8, 0, 1]], device=DEV)
    up = torch.randn(2, 3, 3, generator=gen).to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = layer(tok)
    torch.cuda.current_stream().wait_stream(side)
    (d,) = torch.autograd.grad(z, [layer.weight], up)
    w = layer.weight.detach().double().cpu()
    for v in (0, 1, 2, 4, 8):
        for k in range(3):
            hi, lo = w.clone(), w.clone()
            hi[v, k] += 1e-6
            lo[v, k] -= 1e-6
            diff = ((torch.exp(1 - 0.8 * hi) - torch.exp(1 - 0.8 * lo))[tok.cpu()] * up.double().cpu()).sum() / 2e-6
            # differences: 1e-12 of the third derivative, 1e-16 / 1e-6 of rounding; the kernel: a dozen roundings of terms below 30
            assert abs(float(d[v, k]) - float(diff)) < 1e-4
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z = layer(tok)
        with torch.no_grad():
            layer.weight.add_(1.0)
        z.sum().backward()
