"""The scaled embedding lookup and the table's gradient by sorted tokens (bfb_embed_scaled, bfb_embed_scaled_bwd) against the
definitions in 64 bits.

A lookup multiplies once and rounds once. A gradient row is a sum of n fp32 terms, off by at most n u sum |dout| (u = 2^-24)
whatever the order, then multiplied, then rounded to the table's format (half a step: 2^-24 or 2^-8)."""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = ["f32", "bf16"]


def types(torch, name):
    return torch.float32 if name == "f32" else torch.bfloat16


def half(t):
    return U if "32" in str(t) else 2.0 ** -8


def code(gpu, t):
    return gpu.F32 if "32" in str(t) else gpu.BF16


def gradient(gpu, torch, ids, dout, vocab, dim, table_dtype, scale, into=None, stream=None, ws=None):
    tokens = ids.numel()
    if ws is None:
        n = C.c_size_t(0)
        gpu.check(gpu.lib().bfb_embed_scaled_bwd_workspace(tokens, vocab, dim, C.byref(n)))
        ws = torch.full((max(1, n.value),), 0x7F, dtype=torch.uint8, device="cuda")
    whole = torch.full((vocab + 1, dim), 9.0, dtype=table_dtype, device="cuda")
    if into is not None:
        whole[:vocab] = into
    gpu.check(gpu.lib().bfb_embed_scaled_bwd(ids.data_ptr(), dout.data_ptr(), code(gpu, dout.dtype), max(dim, dout.stride(0)), whole.data_ptr(),
                                             code(gpu, table_dtype), tokens, vocab, dim, scale, int(into is not None), ws.data_ptr(),
                                             ws.numel(), stream))
    return whole


def check_gradient(torch, whole, ids, dout, vocab, scale, into=None):
    ok = (ids >= 0) & (ids < vocab)
    at = ids[ok].long()
    d = dout[ok].double()
    want = torch.zeros(vocab, dout.shape[1], dtype=torch.float64, device="cuda").index_add_(0, at, d)
    mass = torch.zeros_like(want).index_add_(0, at, d.abs())
    n = torch.zeros(vocab, dtype=torch.float64, device="cuda").index_add_(0, at, torch.ones_like(at, dtype=torch.float64))
    s = float(torch.tensor(scale, dtype=torch.float32))
    want, err = want * s, (n[:, None] + 2) * U * mass * abs(s)
    if into is not None:
        want = want + into.double()
        err = err + 2 * U * want.abs()
        assert torch.equal(whole[:vocab][n == 0], into[n == 0])
    got = whole[:vocab].double()
    assert bool(((got - want).abs() <= err + half(whole.dtype) * (want.abs() + err) + 1e-37).all())
    assert (whole[vocab] == 9.0).all()


@pytest.mark.parametrize("tokens,vocab,dim", [(1, 1, 1), (3, 7, 5), (128, 256, 64), (257, 50, 33), (1000, 70001, 24), (40, 33, 1028)])
@pytest.mark.parametrize("table,out", [(a, b) for a in TYPES for b in TYPES])
@pytest.mark.parametrize("pad", [0, 8])
def test_lookup(gpu, tokens, vocab, dim, table, out, pad):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(tokens + dim)
    t = torch.randn(vocab, dim, generator=gen, device="cuda").to(types(torch, table))
    ids = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda").float()
    bad = torch.tensor([-1.0, float(vocab), float("nan"), float("inf"), 3e9], device="cuda")[:tokens // 2]
    ids[:bad.numel()] = bad
    whole = torch.full((tokens + 1, dim + pad), 9.0, dtype=types(torch, out), device="cuda")
    count = torch.zeros(1, dtype=torch.int32, device="cuda")
    gpu.check(gpu.lib().bfb_embed_scaled(ids.data_ptr(), t.data_ptr(), code(gpu, t.dtype), whole.data_ptr(), code(gpu, whole.dtype), dim + pad,
                                         tokens, vocab, dim, 3.25, count.data_ptr(), None))
    torch.cuda.synchronize()
    ok = torch.ones(tokens, dtype=torch.bool, device="cuda")
    ok[:bad.numel()] = False
    want = torch.where(ok[:, None], (t[torch.where(ok, ids, torch.zeros_like(ids)).long()].float() * 3.25).to(whole.dtype), torch.zeros((), device="cuda", dtype=whole.dtype))
    assert torch.equal(whole[:tokens, :dim], want) and int(count) == bad.numel()
    assert (whole[tokens:] == 9.0).all() and (whole[:, dim:] == 9.0).all()


@pytest.mark.parametrize("tokens,vocab,dim", [(1, 1, 1), (1, 1000, 64), (7, 3, 5), (8, 8, 16), (9, 2, 128), (31, 300, 33), (300, 64, 1028), (2500, 40, 8),
                                              (4096, 100, 260), (4097, 513, 40), (10000, 70001, 17), (70000, 12, 24)])
@pytest.mark.parametrize("dout_type,table_type", [(a, b) for a in TYPES for b in TYPES])
def test_gradient(gpu, tokens, vocab, dim, dout_type, table_type):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(tokens + vocab + dim)
    # frequencies that fall with the rank: one id has a large share of the tokens
    u = torch.rand(tokens, generator=gen, device="cuda")
    ids = (torch.floor(torch.exp(u * torch.log(torch.tensor(vocab + 1.0)))) - 1.0).clamp_(0, vocab - 1)
    dout = torch.randn(tokens, dim, generator=gen, device="cuda").to(types(torch, dout_type))
    whole = gradient(gpu, torch, ids, dout, vocab, dim, types(torch, table_type), 1.5)
    again = gradient(gpu, torch, ids, dout, vocab, dim, types(torch, table_type), 1.5)
    torch.cuda.synchronize()
    check_gradient(torch, whole, ids, dout, vocab, 1.5)
    assert torch.equal(whole, again)


@pytest.mark.parametrize("name", ["one id", "ascending", "descending", "borders", "no id", "half without"])
@pytest.mark.parametrize("tokens,dim", [(5000, 64), (40, 7), (70000, 16)])
def test_gradient_of_arranged_ids(gpu, name, tokens, dim):
    """Runs as long as the list, of one entry, that end on and beside the borders of pieces, and tokens that name no row."""
    import torch
    vocab = 5000
    i = torch.arange(tokens, device="cuda")
    ids = {"one id": torch.full((tokens,), 77), "ascending": i % vocab, "descending": vocab - 1 - i % vocab, "borders": i // 64 % vocab,
           "no id": torch.full((tokens,), -1), "half without": torch.where(i % 2 == 0, i % 9, torch.full_like(i, vocab))}[name].float().cuda()
    dout = torch.randn(tokens, dim, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    whole = gradient(gpu, torch, ids, dout, vocab, dim, torch.float32, 1.0)
    torch.cuda.synchronize()
    check_gradient(torch, whole, ids, dout, vocab, 1.0)


@pytest.mark.parametrize("table_type", TYPES)
@pytest.mark.parametrize("tokens,vocab,dim", [(5, 900, 64), (3000, 70, 36), (3000, 70, 35)])
def test_gradient_added_to_what_is_there(gpu, table_type, tokens, vocab, dim):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(8)
    t = types(torch, table_type)
    into = torch.randn(vocab, dim, generator=gen, device="cuda").to(t)
    ids = torch.randint(0, vocab // 2, (tokens,), generator=gen, device="cuda").float()
    wide = torch.randn(tokens, dim + 4, generator=gen, device="cuda")
    whole = gradient(gpu, torch, ids, wide[:, :dim], vocab, dim, t, -0.5, into=into)
    torch.cuda.synchronize()
    check_gradient(torch, whole, ids, wide[:, :dim], vocab, -0.5, into=into)


def test_gradient_in_a_graph_and_with_no_tokens(gpu):
    import torch
    tokens, vocab, dim = 6000, 300, 40
    gen = torch.Generator(device="cuda").manual_seed(12)
    ids = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda").float()
    dout = torch.randn(tokens, dim, generator=gen, device="cuda")
    n = C.c_size_t(0)
    gpu.check(gpu.lib().bfb_embed_scaled_bwd_workspace(tokens, vocab, dim, C.byref(n)))
    ws = torch.empty(n.value, dtype=torch.uint8, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        out = gradient(gpu, torch, ids, dout, vocab, dim, torch.float32, 2.0, stream=torch.cuda.current_stream().cuda_stream, ws=ws)
    ids.copy_(torch.randint(0, vocab, (tokens,), generator=gen, device="cuda").float())
    graph.replay()
    want = gradient(gpu, torch, ids, dout, vocab, dim, torch.float32, 2.0)
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    empty = gradient(gpu, torch, ids[:0], dout[:0], vocab, dim, torch.float32, 2.0)
    kept = gradient(gpu, torch, ids[:0], dout[:0], vocab, dim, torch.float32, 2.0, into=want[:vocab])
    torch.cuda.synchronize()
    assert (empty[:vocab] == 0).all() and torch.equal(kept[:vocab], want[:vocab])


def test_tied_table_step(gpu):
    """The two ends of a decoder with a tied table run together: lookup, loss, the head's gradient into dE, the lookup's gradient
    added to it; the slope of the loss along a direction of the table agrees with it."""
    import torch
    tokens, vocab, dim, scale = 96, 150, 40, 1.5
    gen = torch.Generator(device="cuda").manual_seed(21)
    table = torch.randn(vocab, dim, generator=gen, device="cuda") * 0.3
    ids = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda").float()
    labels = torch.roll(ids, -1)
    labels[-1] = -1
    lib = gpu.lib()
    n = C.c_size_t(0)
    gpu.check(lib.bfb_linear_cross_entropy_workspace(gpu.F32, tokens, vocab, dim, 1, C.byref(n)))
    ws = torch.empty(n.value, dtype=torch.uint8, device="cuda")
    x, loss, lse, summary = torch.empty(tokens, dim, device="cuda"), torch.empty(tokens, device="cuda"), torch.empty(tokens, device="cuda"), torch.empty(3, device="cuda")

    def run(e):
        gpu.check(lib.bfb_embed_scaled(ids.data_ptr(), e.data_ptr(), gpu.F32, x.data_ptr(), gpu.F32, dim, tokens, vocab, dim, scale, None, None))
        gpu.check(lib.bfb_linear_cross_entropy_fwd(x.data_ptr(), dim, e.data_ptr(), dim, None, labels.data_ptr(), loss.data_ptr(), lse.data_ptr(),
                                                   summary.data_ptr(), gpu.F32, tokens, vocab, dim, None, ws.data_ptr(), ws.numel(), None, None))
        torch.cuda.synchronize()
        return float(loss.double().sum()) / float(summary[1])
    run(table)
    dx, de = torch.empty_like(x), torch.empty_like(table)
    gpu.check(lib.bfb_linear_cross_entropy_bwd(x.data_ptr(), dim, table.data_ptr(), dim, None, labels.data_ptr(), lse.data_ptr(), None,
                                               summary.data_ptr() + 8, 1.0, dx.data_ptr(), dim, de.data_ptr(), dim, None, gpu.F32, gpu.F32, tokens,
                                               vocab, dim, ws.data_ptr(), ws.numel(), None, None))
    whole = gradient(gpu, torch, ids, dx, vocab, dim, torch.float32, scale, into=de)
    torch.cuda.synchronize()
    e64 = table.double().requires_grad_()
    z = torch.nn.functional.embedding(ids.long(), e64) * scale @ e64.t()
    torch.nn.functional.cross_entropy(z, labels.long(), ignore_index=-1).backward()
    # products of length dim and vocab in fp32: a few hundred roundings of terms of the size of the result's largest
    assert float((whole[:vocab].double() - e64.grad).abs().max()) <= 400 * U * float(e64.grad.abs().max()) + 1e-9
    v = torch.randn(vocab, dim, generator=gen, device="cuda")
    h = 2.0 ** -9
    slope = (run(table + h * v) - run(table - h * v)) / (2 * h)
    want = float((v.double() * whole[:vocab].double()).sum())
    assert abs(slope - want) <= 100 * h * h * (1 + abs(want)) + 5 * 2.0 ** -22 / (2 * h)
