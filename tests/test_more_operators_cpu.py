"""Refusals of the head, embedding, norm and balance entry points that need no GPU (nothing is launched: arguments are
checked before any HIP call; addresses are made up), and what their plans promise."""
import ctypes

import pytest
import torch

ARG, ALIGN, WORKSPACE, OVERLAP = 1001, 1002, 1004, 1005
A, B, C, D, E, F, G, W = (i << 40 for i in range(1, 9))
BIG = 1 << 38


@pytest.fixture(scope="module")
def lib():
    from muon_sr_amd import _lib
    return _lib.lib()


def test_head_sizes(lib):
    f, b = ctypes.c_size_t(), ctypes.c_size_t()
    plan = (ctypes.c_int32 * 7)()
    for rows, vocab, d in ((0, 1, 8), (1, 1, 8), (7, 512, 256), (4096, 16384, 384), (8192, 128256, 4096), (100000, 50257, 1024),
                           (1 << 22, 1 << 17, 64), (1, (1 << 24) - 1, 8)):
        assert lib.msr_head_workspace_bytes(rows, vocab, d, ctypes.byref(f), ctypes.byref(b)) == 0
        assert lib.msr_head_plan(rows, vocab, d, plan) == 0
        fwd, logits, dx, dxs, dw, dws, piece = plan
        assert {fwd, logits, dx, dw} <= {64, 128, 256} and 1 <= dxs <= 16 and 1 <= dws <= 16
        assert 0 < piece <= max(8, (vocab + 7) // 8 * 8) and (piece % 256 == 0 or piece >= vocab)
        assert f.value >= 8 * rows * -(-vocab // fwd) + 8 * rows
        assert b.value >= 2 * rows * piece + 4 * dxs * rows * d + (4 * dws * piece * d if dws > 1 else 0)
        # neither grows with rows x words: a piece of G is 512 MiB, or 256 words of every row
        assert 2 * rows * piece <= max(512 << 20, 2 * 256 * rows)
    for rows, vocab, d in ((-1, 5, 8), (1 << 24, 5, 8), (5, 0, 8), (5, 1 << 24, 8), (5, 5, 0), (5, 5, 12), (5, 5, 1 << 17), ((1 << 23), 1 << 23, 8)):
        assert lib.msr_head_workspace_bytes(rows, vocab, d, ctypes.byref(f), ctypes.byref(b)) == ARG
        assert lib.msr_head_plan(rows, vocab, d, plan) == ARG
    assert lib.msr_head_workspace_bytes(5, 5, 8, None, ctypes.byref(b)) == ARG and lib.msr_head_plan(5, 5, 8, None) == ARG


def test_head_forward(lib):
    def call(x=A, ldx=64, w=B, target=C, i64=1, rows=100, vocab=500, d=64, red=2, packed=D, kept=E, sums=F, loss=G, ws=W, n=BIG):
        return lib.msr_head_forward(x, ldx, w, target, i64, -100, rows, vocab, d, red, packed, kept, sums, loss, ws, n, None)
    for bad in (dict(x=None), dict(w=None), dict(target=None), dict(packed=None), dict(kept=None), dict(sums=None), dict(loss=None), dict(ldx=63),
                dict(red=3), dict(red=-1), dict(rows=-1), dict(vocab=0), dict(d=60)):
        assert call(**bad) == ARG, bad
    for bad in (dict(x=A + 1), dict(w=B + 8), dict(packed=D + 8), dict(target=C + 4), dict(target=C + 2, i64=0), dict(kept=E + 2), dict(sums=F + 4),
                dict(loss=G + 1), dict(ws=W + 8)):
        assert call(**bad) == ALIGN, bad
    assert call(ws=None) == WORKSPACE and call(n=100) == WORKSPACE and b"workspace" in lib.msr_last_error()
    for bad in (dict(packed=A + 64), dict(kept=C), dict(sums=E + 1200), dict(loss=B + 64), dict(ws=A), dict(ws=D + 16), dict(loss=F + 4), dict(packed=B)):
        assert call(**bad) == OVERLAP, bad
    assert call(rows=(1 << 24) - 1, vocab=1 << 16, d=64) == ARG and b"tiles" in lib.msr_last_error()


def test_head_backward(lib):
    def call(packed=A, w=B, kept=C, sums=D, dloss=E, rows=100, vocab=500, d=64, red=2, dx=F, dw=G, mode=-1, seed=0, zero=0, inject=None, ws=W, n=BIG):
        return lib.msr_head_backward(packed, w, kept, sums, dloss, rows, vocab, d, red, dx, dw, mode, seed, zero, inject, ws, n, None)
    for bad in (dict(packed=None), dict(w=None), dict(kept=None), dict(sums=None), dict(dloss=None), dict(red=5), dict(mode=3), dict(mode=-2),
                dict(mode=2), dict(d=65)):
        assert call(**bad) == ARG, bad
    for bad in (dict(packed=A + 8), dict(w=B + 2), dict(dx=F + 8), dict(dw=G + 4), dict(kept=C + 1), dict(sums=D + 4), dict(dloss=E + 2), dict(ws=W + 4)):
        assert call(**bad) == ALIGN, bad
    assert call(n=1000) == WORKSPACE
    for bad in (dict(dx=A), dict(dw=B), dict(dx=G + 64), dict(ws=G), dict(dw=C - 64), dict(dx=E), dict(dw=A + 64), dict(mode=2, inject=G + 64)):
        assert call(**bad) == OVERLAP, bad
    assert call(dx=None, dw=None) == 0            # nothing wanted


def test_embedding(lib):
    look = lambda ids=A, i64=1, n=10, w=B, vocab=50, d=16, y=C, elem=0: lib.msr_embedding(ids, i64, n, w, vocab, d, 1.0, y, elem, None)  # noqa: E731
    assert look(n=0) == 0 and look(d=0) == 0
    for bad in (dict(ids=None), dict(w=None), dict(y=None), dict(n=-1), dict(n=1 << 28), dict(vocab=0), dict(vocab=1 << 27), dict(d=-1), dict(elem=2)):
        assert look(**bad) == ARG, bad
    assert look(ids=A + 4) == ALIGN and look(w=B + 1) == ALIGN and look(y=C + 2, elem=1) == ALIGN
    assert look(y=A) == OVERLAP and look(y=B + 32) == OVERLAP
    size = ctypes.c_size_t()
    assert lib.msr_embedding_workspace_bytes(2000, 50, 16, ctypes.byref(size)) == 0 and size.value >= 16000 + 32 * 2 * 64
    assert lib.msr_embedding_workspace_bytes(100, 50, 16, ctypes.byref(size)) == 0 and size.value == 0
    assert lib.msr_embedding_workspace_bytes(100, 50, 16, None) == ARG and lib.msr_embedding_workspace_bytes(-1, 50, 16, ctypes.byref(size)) == ARG

    def grad(ids=A, i64=1, n=2000, dy=B, ld=16, vocab=50, d=16, dw=C, elem=0, ws=W, size=BIG):
        return lib.msr_embedding_grad(ids, i64, n, dy, ld, vocab, d, 1.0, -1, dw, elem, ws, size, None)

    def accum(ids=A, n=2000, dy=B, ld=16, vocab=50, d=16, acc=C, mode=1, inject=None, ws=W, size=BIG):
        return lib.msr_embedding_grad_sr_accum(ids, 1, n, dy, ld, vocab, d, 1.0, -1, acc, 7, 0, mode, inject, ws, size, None)
    assert grad(d=0, ld=0) == 0
    for bad in (dict(ids=None), dict(dy=None), dict(dw=None), dict(ld=15), dict(n=1 << 28), dict(vocab=1 << 27), dict(elem=3)):
        assert grad(**bad) == ARG, bad
    assert grad(dy=B + 1) == ALIGN and grad(dw=C + 2, elem=1) == ALIGN and grad(ws=W + 4) == ALIGN
    assert grad(ws=None) == WORKSPACE and grad(size=64) == WORKSPACE
    assert grad(dw=A) == OVERLAP and grad(dw=B + 64) == OVERLAP and grad(ws=B) == OVERLAP and grad(ws=C) == OVERLAP
    assert grad(vocab=(1 << 27) - 1, d=1 << 14, ld=1 << 14, dw=1 << 50) == ARG and b"launch" in lib.msr_last_error()
    assert grad(n=500, vocab=(1 << 27) - 1, d=1 << 12, ld=1 << 12, dw=1 << 50) == ARG and b"launch" in lib.msr_last_error()
    for bad in (dict(mode=-1), dict(mode=3), dict(mode=2)):
        assert accum(**bad) == ARG, bad
    assert accum(mode=2, inject=C + 64) == OVERLAP


def test_layer_norm(lib):
    def norm(x=A, ld=32, w=B, b=C, rows=10, d=32, y=D, mean=E, rstd=F, elem=0, welem=1):
        return lib.msr_layer_norm(x, ld, w, b, 1e-5, rows, d, y, mean, rstd, elem, welem, None)
    assert norm(rows=0) == 0 and norm(d=0) == 0
    for bad in (dict(x=None), dict(y=None), dict(mean=None), dict(rstd=None), dict(ld=31), dict(rows=-1), dict(d=(1 << 24) + 1), dict(elem=2), dict(welem=-1)):
        assert norm(**bad) == ARG, bad
    assert norm(x=A + 1) == ALIGN and norm(w=B + 2) == ALIGN and norm(mean=E + 2) == ALIGN and norm(y=D + 2, elem=1) == ALIGN
    assert norm(y=A) == OVERLAP and norm(y=A + 64) == OVERLAP and norm(mean=E, rstd=E + 4) == OVERLAP and norm(rstd=B) == OVERLAP
    size = ctypes.c_size_t()
    assert lib.msr_layer_norm_workspace_bytes(10, 32, 0, ctypes.byref(size)) == 0 and size.value >= 256
    assert lib.msr_layer_norm_workspace_bytes(10, 32, 7, ctypes.byref(size)) == ARG and lib.msr_layer_norm_workspace_bytes(10, 32, 0, None) == ARG

    def grad(dy=A, x=B, w=C, mean=D, rstd=E, rows=10, d=32, dx=F, dw=G, db=G + 4096, ldy=32, ldx=32, elem=0, ws=W, n=BIG):
        return lib.msr_layer_norm_grad(dy, ldy, x, ldx, w, mean, rstd, rows, d, dx, dw, db, elem, 1, ws, n, None)
    assert grad(d=0) == 0 and grad(dx=None, dw=None, db=None) == 0
    for bad in (dict(dy=None), dict(x=None), dict(mean=None), dict(rstd=None), dict(ldy=31), dict(ldx=31)):
        assert grad(**bad) == ARG, bad
    assert grad(dx=F + 1) == ALIGN and grad(dw=G + 2) == ALIGN and grad(ws=W + 2) == ALIGN
    assert grad(ws=None) == WORKSPACE and grad(n=16) == WORKSPACE
    assert grad(dx=A) == OVERLAP and grad(dx=B + 64) == OVERLAP and grad(dw=G, db=G + 64) == OVERLAP and grad(ws=F) == OVERLAP and grad(dw=C) == OVERLAP


def test_balance(lib):
    size = ctypes.c_size_t()
    assert lib.msr_balance_workspace_bytes(100, 8, ctypes.byref(size)) == 0 and size.value >= 4 * 17
    assert lib.msr_balance_workspace_bytes(100, 1025, ctypes.byref(size)) == ARG and lib.msr_balance_workspace_bytes(100, 8, None) == ARG

    def loss(logits=A, ld=8, ids=B, i64=1, mask=C, tokens=100, experts=8, k=2, out=D, counts=E, lse=F, slope=G, elem=1, ws=W, n=BIG):
        return lib.msr_balance_loss(logits, ld, ids, i64, mask, tokens, experts, k, out, counts, lse, slope, elem, ws, n, None)
    for bad in (dict(logits=None), dict(ids=None), dict(out=None), dict(counts=None), dict(lse=None), dict(slope=None), dict(ld=7), dict(k=0),
                dict(experts=0), dict(experts=1025), dict(tokens=-1), dict(tokens=1 << 29, k=2), dict(elem=2)):
        assert loss(**bad) == ARG, bad
    assert loss(logits=A + 2) == ALIGN and loss(ids=B + 4) == ALIGN and loss(counts=E + 2) == ALIGN and loss(ws=W + 1) == ALIGN
    assert loss(ws=None) == WORKSPACE and loss(n=8) == WORKSPACE
    assert loss(out=A) == OVERLAP and loss(lse=B + 8) == OVERLAP and loss(ws=C) == OVERLAP and loss(counts=G, slope=G + 16) == OVERLAP
    grad = lambda logits=A, mask=None, lse=B, slope=C, up=D, out=E, tokens=100, elem=1: lib.msr_balance_grad(  # noqa: E731
        logits, 8, mask, lse, slope, up, tokens, 8, out, elem, None)
    assert grad(tokens=0) == 0
    assert grad(logits=None) == ARG and grad(lse=None) == ARG and grad(slope=None) == ARG and grad(up=None) == ARG and grad(out=None) == ARG
    assert grad(out=E + 2) == ALIGN and grad(out=A) == OVERLAP and grad(out=B) == OVERLAP and grad(out=D - 8) == OVERLAP


def test_python_needs_a_gpu():
    import muon_sr_amd as M
    x, w = torch.zeros((4, 16), dtype=torch.bfloat16), torch.zeros((9, 16), dtype=torch.bfloat16)
    ids = torch.zeros(4, dtype=torch.int64)
    head, table, norm = M.SRHead(16, 9), M.SREmbedding(9, 16, padding_idx=2, scale=4.0), M.LayerNorm(16)
    for call in (lambda: M.linear_cross_entropy(x, w, ids), lambda: head.loss(x, ids), lambda: M.embedding(ids, w), lambda: table(ids),
                 lambda: M.embedding_grad_sr_accum(w, ids, x), lambda: M.layer_norm(x), lambda: norm(x),
                 lambda: M.balance_loss(x, ids[:, None])):
        with pytest.raises(ValueError, match="GPU"):
            call()
    # the modules' states are torch's
    assert set(head.state_dict()) == {"weight"} and set(table.state_dict()) == {"weight"} and set(norm.state_dict()) == {"weight", "bias"}
    assert head.weight.shape == (9, 16) and head.weight.dtype == table.weight.dtype == torch.bfloat16 and not table.weight[2].any()


def test_hooks_of_the_head_see_its_loss():
    """A loss is a call of the module: its pre-hooks run before the arguments are checked (here: that they are on a GPU), with the loss's
    arguments; torch.nn.utils.weight_norm's computes the weight.  A subclass whose forward takes x alone keeps its loss."""
    import muon_sr_amd as M
    x, ids = torch.zeros((4, 16), dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int64)
    head, seen = M.SRHead(16, 9), []
    torch.nn.utils.weight_norm(head)
    head.register_forward_pre_hook(lambda module, args: seen.append(args))
    with torch.no_grad():
        head.weight_g.mul_(2)
    before = head.weight.clone()
    with pytest.raises(ValueError, match="GPU"):
        head.loss(x, ids, reduction="sum")
    (args,) = seen
    assert args[0] is x and args[1] is ids and args[2:] == (-100, "sum")
    assert torch.equal(head.weight, 2 * before)

    class Last(M.SRHead):
        def forward(self, x):
            return super().forward(x[-1:])
    last = Last(16, 9)
    assert last(x).shape == (1, 9)
    with pytest.raises(ValueError, match="GPU"):
        last.loss(x, ids)
    with pytest.raises(TypeError):
        head.loss(x, None)


def test_embedding_from_pretrained():
    """As nn.Embedding's: the weight is the given tensor, frozen unless asked; options that are not taken are refused."""
    import muon_sr_amd as M
    for dtype in (torch.bfloat16, torch.float32):
        table = torch.randn((9, 16)).to(dtype)
        m = M.SREmbedding.from_pretrained(table)
        theirs = torch.nn.Embedding.from_pretrained(table)
        assert isinstance(m, M.SREmbedding) and m.weight.data_ptr() == table.data_ptr() and not m.weight.requires_grad
        assert (m.num_embeddings, m.embedding_dim, m.padding_idx) == (theirs.num_embeddings, theirs.embedding_dim, theirs.padding_idx)
        m = M.SREmbedding.from_pretrained(table, False, -1, scale=4.0)
        assert m.weight.requires_grad and m.weight.is_leaf and m.padding_idx == 8 and m.scale == 4.0
        assert torch.equal(m.weight, table) and m.state_dict().keys() == theirs.state_dict().keys()
    with pytest.raises(ValueError, match="vocab"):
        M.SREmbedding.from_pretrained(table[0])
    for bad in (dict(max_norm=1.0), dict(sparse=True)):
        with pytest.raises(TypeError):
            M.SREmbedding.from_pretrained(table, **bad)
