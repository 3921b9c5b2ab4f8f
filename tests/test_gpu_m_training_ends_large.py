"""The training-side operators at the ends of a decoder where offsets pass 2^31 elements, and with gradients whose rows the tensor-core
route cannot store. Bounds as in the operators' own tests: half a step of the result's format plus the counted fp32 roundings."""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def workspace(gpu, torch, query, *args):
    n = C.c_size_t(0)
    gpu.check(getattr(gpu.lib(), query)(*args, C.byref(n)))
    return torch.empty(max(1, n.value), dtype=torch.uint8, device="cuda")


def test_embedding_table_beyond_32_bits(gpu):
    import torch
    vocab, dim, tokens = 2_200_000, 1000, 300
    gen = torch.Generator(device="cuda").manual_seed(1)
    table = torch.empty(vocab, dim, device="cuda").normal_(generator=gen)
    ids = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda").float()
    ids[:4] = torch.tensor([0.0, vocab - 1.0, vocab - 1.0, vocab - 2.0], device="cuda")
    out = torch.empty(tokens, dim, device="cuda")
    lib = gpu.lib()
    gpu.check(lib.bfb_embed_scaled(ids.data_ptr(), table.data_ptr(), gpu.F32, out.data_ptr(), gpu.F32, dim, tokens, vocab, dim, 2.0, None, None))
    torch.cuda.synchronize()
    assert torch.equal(out, table[ids.long()] * 2.0)
    dtable = table.fill_(7.0)
    ws = workspace(gpu, torch, "bfb_embed_scaled_bwd_workspace", tokens, vocab, dim)
    gpu.check(lib.bfb_embed_scaled_bwd(ids.data_ptr(), out.data_ptr(), gpu.F32, dim, dtable.data_ptr(), gpu.F32, tokens, vocab, dim, 0.5, 0,
                                       ws.data_ptr(), ws.numel(), None))
    torch.cuda.synchronize()
    rows, where = torch.unique(ids.long(), return_inverse=True)
    want = torch.zeros(len(rows), dim, dtype=torch.float64, device="cuda").index_add_(0, where, out.double()) * 0.5
    mass = torch.zeros(len(rows), dim, dtype=torch.float64, device="cuda").index_add_(0, where, out.double().abs())
    assert bool(((dtable[rows].double() - want).abs() <= (tokens + 2) * U * mass).all())
    dtable[rows] = 0.0
    assert int(torch.count_nonzero(dtable)) == 0


def test_distillation_logits_beyond_32_bits(gpu):
    import torch
    rows, vocab = 11000, 200003
    z = torch.empty(rows, vocab, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(2))
    some = [0, 5000, rows - 1]
    kept = z[some].double()
    ids = torch.tensor([[3.0, vocab - 1.0]], device="cuda").repeat(rows, 1)
    teacher = torch.tensor([[1.0, 2.0]], device="cuda").repeat(rows, 1)
    loss = torch.empty(rows, device="cuda")
    gpu.check(gpu.lib().bfb_distill_topk(z.data_ptr(), gpu.BF16, vocab, ids.data_ptr(), teacher.data_ptr(), gpu.F32, 2, 1.0, None, None, 1.0,
                                         loss.data_ptr(), None, z.data_ptr(), gpu.BF16, vocab, rows, vocab, None, None))
    torch.cuda.synchronize()
    log_p = torch.log_softmax(kept, 1)
    q = torch.softmax(teacher[0].double(), 0)
    at = ids[0].long()
    want = (q * (q.log() - log_p[:, at])).sum(1)
    rel = (8 * 104 + 64) * U
    assert float((loss[some].double() - want).abs().max()) <= rel * 40
    p = log_p.exp()
    grad = p.clone()
    grad[:, at] -= q
    assert bool(((z[some].double() - grad).abs() <= rel * (p + grad.abs()) + 2.0 ** -8 * grad.abs() * (1 + rel) + 1e-37).all())
    assert bool(loss.isfinite().all())


def test_hidden_states_beyond_32_bits(gpu):
    import torch
    tokens, vocab, dim = 1_100_000, 300, 2048
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.empty(tokens, dim, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    w = (torch.randn(vocab, dim, generator=gen, device="cuda") * (2.0 / dim ** 0.5)).bfloat16()
    labels = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda").float()
    lib = gpu.lib()
    ws = workspace(gpu, torch, "bfb_linear_cross_entropy_workspace", gpu.BF16, tokens, vocab, dim, 1)
    loss, lse, summary = torch.empty(tokens, device="cuda"), torch.empty(tokens, device="cuda"), torch.empty(3, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    gpu.check(lib.bfb_linear_cross_entropy_fwd(x.data_ptr(), dim, w.data_ptr(), dim, None, labels.data_ptr(), loss.data_ptr(), lse.data_ptr(),
                                               summary.data_ptr(), gpu.BF16, tokens, vocab, dim, None, ws.data_ptr(), ws.numel(),
                                               status.data_ptr(), None))
    dx, dw = torch.empty_like(x), torch.empty(vocab, dim, device="cuda")
    db = torch.empty(vocab, device="cuda")
    # two calls: dx is bf16, dW fp32
    for grads, code in (((dx.data_ptr(), dim, None, dim, db.data_ptr()), gpu.BF16), ((None, dim, dw.data_ptr(), dim, None), gpu.F32)):
        gpu.check(lib.bfb_linear_cross_entropy_bwd(x.data_ptr(), dim, w.data_ptr(), dim, None, labels.data_ptr(), lse.data_ptr(), None, None, 1.0,
                                                   *grads, gpu.BF16, code, tokens, vocab, dim, ws.data_ptr(), ws.numel(), status.data_ptr(), None))
    torch.cuda.synchronize()
    assert int(status) == 0 and float(summary[1]) == tokens
    w64 = w.double()
    want_dw = torch.zeros(vocab, dim, dtype=torch.float64, device="cuda")
    mass = torch.zeros_like(want_dw)
    want_db = torch.zeros(vocab, dtype=torch.float64, device="cuda")
    for begin in range(0, tokens, 100_000):
        part = slice(begin, min(tokens, begin + 100_000))
        x64 = x[part].double()
        z = x64 @ w64.t()
        l64 = torch.logsumexp(z, 1)
        at = labels[part].long()
        rows = torch.arange(len(at), device="cuda")
        # logits: 2 dim roundings of terms that sum to at most |x| |w| (Cauchy), lse and loss two of them
        z_err = 2 * dim * U * float(x64.norm(dim=1).max() * w64.norm(dim=1).max()) + 64 * U
        assert float((loss[part].double() - (l64 - z[rows, at])).abs().max()) <= 3 * z_err
        dz = torch.exp(z - l64[:, None])
        dz[rows, at] -= 1.0
        want_dw += dz.t() @ x64
        mass += dz.abs().t() @ x64.abs()
        want_db += dz.sum(0)
        got = dx[part].double()
        want = dz @ w64
        err = (2.0 ** -8 + 3 * z_err + 2 * vocab * U) * (dz.abs() @ w64.abs())
        assert bool(((got - want).abs() <= err + 2.0 ** -8 * (want.abs() + err)).all())
        del z, dz, got, want, err, x64
    # the fp32 sum of one part of a split reduction: a sixteenth of the rows, in truncated additions
    assert bool(((dw.double() - want_dw).abs() <= (2.0 ** -8 + 3 * z_err + 2 * (tokens / 16 + 64) * U) * mass).all())
    assert float((db.double() - want_db).abs().max()) <= (3 * z_err + 4096 * U) * tokens


@pytest.mark.parametrize("ld,offset", [(65, 0), (72, 1)])
def test_gradients_on_rows_tma_could_not_store(gpu, ld, offset):
    """Operands for the tensor cores, results at an odd pitch or address: the CUDA cores take the backward."""
    import torch
    tokens, vocab, dim = 150, 400, 64
    gen = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(tokens, dim, generator=gen, device="cuda").bfloat16()
    w = (torch.randn(vocab, dim, generator=gen, device="cuda") * 0.25).bfloat16()
    labels = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda").float()
    lib = gpu.lib()
    ws = workspace(gpu, torch, "bfb_linear_cross_entropy_workspace", gpu.BF16, tokens, vocab, dim, 1)
    lse = torch.empty(tokens, device="cuda")
    gpu.check(lib.bfb_linear_cross_entropy_fwd(x.data_ptr(), dim, w.data_ptr(), dim, None, labels.data_ptr(), None, lse.data_ptr(), None, gpu.BF16,
                                               tokens, vocab, dim, None, ws.data_ptr(), ws.numel(), None, None))
    dx, dw = (torch.full(((n + 1) * ld + 8,), 5.0, dtype=torch.bfloat16, device="cuda") for n in (tokens, vocab))
    gpu.check(lib.bfb_linear_cross_entropy_bwd(x.data_ptr(), dim, w.data_ptr(), dim, None, labels.data_ptr(), lse.data_ptr(), None, None, 1.0,
                                               dx.data_ptr() + 2 * offset, ld, dw.data_ptr() + 2 * offset, ld, None, gpu.BF16, gpu.BF16, tokens,
                                               vocab, dim, ws.data_ptr(), ws.numel(), None, None))
    torch.cuda.synchronize()
    z = x.double() @ w.double().t()
    dz = torch.softmax(z, 1)
    dz[torch.arange(tokens), labels.long()] -= 1.0
    for got, want, mass in ((dx, dz @ w.double(), dz.abs() @ w.double().abs()), (dw, dz.t() @ x.double(), dz.abs().t() @ x.double().abs())):
        whole = got[offset:offset + want.shape[0] * ld].view(-1, ld)
        err = 2.0 ** -14 * mass   # logits of a few units in fp32 products of depth 64, sums of up to 400 terms
        assert bool(((whole[:, :dim].double() - want).abs() <= err + 2.0 ** -8 * (want.abs() + err)).all())
        assert (whole[:, dim:] == 5.0).all() and (got[:offset] == 5.0).all() and (got[offset + want.shape[0] * ld:] == 5.0).all()
