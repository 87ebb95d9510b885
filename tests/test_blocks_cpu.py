"""Operators over blocks without a GPU: public names, checks made before any launch,
and the C entry points' refusals."""

import ctypes
import inspect

import pytest
import torch

import flagsparse_amd as fs
from flagsparse_amd import _lib, blocks

NAMES = {
    "PreparedBlockSequences", "prepare_block_sequences", "flagsparse_block_means", "flagsparse_block_select",
    "flagsparse_block_attention", "flagsparse_block_attention_grad",
}
FAKE = 4096  # an address that no refused call reads


def test_public_names():
    assert NAMES <= set(fs.__all__) and NAMES <= set(dir(fs))
    for name in NAMES:
        assert inspect.getdoc(getattr(fs, name))


def test_sequences_are_checked():
    i32 = torch.zeros(3, dtype=torch.int32)
    prepare = fs.prepare_block_sequences
    with pytest.raises(ValueError, match="block_size must be one of"):
        prepare(48, i32, k_offsets=i32)
    with pytest.raises(ValueError, match="either k_offsets or pages"):
        prepare(64, i32)
    with pytest.raises(ValueError, match="either k_offsets or pages"):
        prepare(64, i32, k_offsets=i32, pages=i32[None])
    with pytest.raises(ValueError, match="k_lengths goes with pages"):
        prepare(64, i32, k_offsets=i32, k_lengths=i32)
    with pytest.raises(ValueError, match="k_lengths must be given"):
        prepare(64, i32, pages=i32[None])
    with pytest.raises(TypeError, match="k_offsets dtype must be torch.int32"):
        prepare(64, i32, k_offsets=i32.long())
    with pytest.raises(TypeError, match="pages dtype must be torch.int32"):
        prepare(64, i32, pages=i32[None].long(), k_lengths=i32[:1])
    with pytest.raises(TypeError, match="k_offsets must be a torch.Tensor"):
        prepare(64, i32, k_offsets=[0, 1])
    with pytest.raises(ValueError, match="q_offsets must have 3 elements"):
        prepare(64, i32[:2], k_offsets=i32)
    with pytest.raises(ValueError, match="at least one element"):
        prepare(64, k_offsets=i32[:0])
    with pytest.raises(ValueError, match="contiguous 1D"):
        prepare(64, k_offsets=torch.zeros(6, dtype=torch.int32)[::2])
    with pytest.raises(ValueError, match="2D tensor of contiguous rows"):
        prepare(64, pages=torch.zeros(4, 4, dtype=torch.int32).t()[:, ::2], k_lengths=torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError, match="q_offsets must be a CUDA tensor"):
        prepare(64, i32, k_offsets=i32)


class _Cuda(torch.Tensor):
    """A CPU tensor that says it is on a GPU: for checks alone."""

    is_cuda = True


def _fake(shape, dtype=torch.float16):
    return torch.zeros(shape, dtype=dtype).as_subclass(_Cuda)


def _seqs(n, paged=False, q_offsets=True):
    i32 = torch.zeros(n + 1, dtype=torch.int32)
    pages = torch.zeros((n, 4), dtype=torch.int32) if paged else None
    return blocks.PreparedBlockSequences(64, i32 if q_offsets else None, None if paged else i32, pages,
                                         i32[:n] if paged else None, n, torch.device("cpu"))


def test_operands_are_checked():
    seqs = _seqs(2)
    q, k = _fake((5, 6, 64)), _fake((40, 3, 64))
    ids = _fake((5, 3, 4), torch.int32)
    attend = fs.flagsparse_block_attention
    with pytest.raises(TypeError, match="seqs must be a PreparedBlockSequences"):
        attend(q, k, k, ids, None)
    with pytest.raises(ValueError, match="k must be a CUDA tensor"):
        attend(q, torch.zeros(40, 3, 64, dtype=torch.float16), k, ids, seqs)
    with pytest.raises(TypeError, match="k dtype must be one of"):
        attend(q, _fake((40, 3, 64), torch.float64), k, ids, seqs)
    with pytest.raises(ValueError, match="k must be a 3D tensor"):
        attend(q, k[0], k, ids, seqs)
    with pytest.raises(ValueError, match="k must be a 4D tensor"):
        attend(q, k, k, ids, _seqs(2, paged=True))
    with pytest.raises(ValueError, match="power of two of rows, at least 16"):
        attend(q, _fake((4, 24, 3, 64)), k, ids, _seqs(2, paged=True))
    with pytest.raises(ValueError, match="width must be a multiple of 8 from 8 to 256, got 36"):
        attend(q, _fake((40, 3, 36)), k, ids, seqs)
    with pytest.raises(ValueError, match="width must be a multiple of 8 from 8 to 128, got 136"):
        attend(q, _fake((40, 3, 136), torch.float32), k, ids, seqs)
    with pytest.raises(TypeError, match="v dtype must match"):
        attend(q, k, _fake((40, 3, 64), torch.bfloat16), ids, seqs)
    with pytest.raises(ValueError, match="v must have k's shape"):
        attend(q, k, k[:39], ids, seqs)
    with pytest.raises(TypeError, match="q dtype must match the keys'"):
        attend(_fake((5, 6, 64), torch.bfloat16), k, k, ids, seqs)
    with pytest.raises(ValueError, match="q must have width 64, got 72"):
        attend(_fake((5, 6, 72)), k, k, ids, seqs)
    with pytest.raises(ValueError, match="q heads must be 1 to 128 times the 3"):
        attend(_fake((5, 7, 64)), k, k, ids, seqs)
    with pytest.raises(ValueError, match="q heads must be 1 to 128 times the 1"):
        attend(_fake((5, 129, 64)), k[:, :1], k[:, :1], ids[:, :1], seqs)
    with pytest.raises(ValueError, match="without q_offsets q must have 2 tokens, got 5"):
        attend(q, k, k, ids, _seqs(2, q_offsets=False))
    with pytest.raises(TypeError, match="blocks dtype must be torch.int32"):
        attend(q, k, k, _fake((5, 3, 4), torch.int64), seqs)
    with pytest.raises(ValueError, match=r"blocks must have shape \(5, 3 or 1, top\)"):
        attend(q, k, k, ids[:, :2], seqs)
    with pytest.raises(ValueError, match="blocks must name 1 to 128 blocks a query, got 129"):
        attend(q, k, k, _fake((5, 3, 129), torch.int32), seqs)
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="scale must be positive and finite"):
            attend(q, k, k, ids, seqs, scale=scale)
    with pytest.raises(ValueError, match="out must be a CUDA tensor"):
        attend(q, k, k, ids, seqs, out=torch.zeros(5, 6, 64, dtype=torch.float16))
    leaf = _fake((5, 6, 64)).requires_grad_()
    with pytest.raises(ValueError, match="out cannot be given where a gradient is recorded"):
        attend(leaf, k, k, ids, seqs, out=_fake((5, 6, 64)))
    with pytest.raises(ValueError, match="keys and values of a cache have no gradient"):
        cache = _fake((4, 16, 3, 64))
        attend(leaf, cache, cache, ids, _seqs(2, paged=True))
    grad = fs.flagsparse_block_attention_grad
    lse = _fake((5, 6), torch.float32)
    with pytest.raises(ValueError, match="groups of up to 96 heads, got 97"):
        wide, keys = _fake((5, 97, 256)), _fake((40, 1, 256))
        grad(wide, wide, keys, keys, ids[:, :1], seqs, wide, _fake((5, 97), torch.float32))
    with pytest.raises(ValueError, match="keys and values of a cache have no gradient"):
        cache = _fake((4, 16, 3, 64))
        grad(q, q, cache, cache, ids, _seqs(2, paged=True), q, lse)
    with pytest.raises(ValueError, match="grad must have q's shape"):
        grad(q[:4], q, k, k, ids, seqs, q, lse)
    with pytest.raises(TypeError, match="out dtype must match q dtype"):
        grad(q, q, k, k, ids, seqs, _fake((5, 6, 64), torch.bfloat16), lse)
    with pytest.raises(TypeError, match="lse dtype must be torch.float32"):
        grad(q, q, k, k, ids, seqs, q, _fake((5, 6)))
    with pytest.raises(ValueError, match=r"lse must have shape \(5, 6\)"):
        grad(q, q, k, k, ids, seqs, q, lse[:, :5])


def test_summaries_and_selection_are_checked():
    seqs = _seqs(2)
    q, k, means = _fake((5, 6, 64)), _fake((40, 3, 64)), _fake((2, 7, 3, 64))
    start = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="out must be given with start"):
        fs.flagsparse_block_means(k, seqs, max_blocks=7, start=start)
    with pytest.raises(ValueError, match="max_blocks must be given without out"):
        fs.flagsparse_block_means(k, seqs)
    with pytest.raises(ValueError, match="out shape/dtype must match result"):
        fs.flagsparse_block_means(k, seqs, out=means[:1])
    with pytest.raises(ValueError, match="out must hold max_blocks blocks, got 7"):
        fs.flagsparse_block_means(k, seqs, max_blocks=6, out=means)
    with pytest.raises(TypeError, match="start dtype must be torch.int32"):
        fs.flagsparse_block_means(k, seqs, start=start.long(), out=means)
    select = fs.flagsparse_block_select
    with pytest.raises(ValueError, match="means must hold 2 sequences' blocks"):
        select(q, means[:1], seqs, 4)
    with pytest.raises(ValueError, match="top must be in 1..128, got 129"):
        select(q, means, seqs, 129)
    for first, recent in ((-1, 1), (0, 0), (2, 3)):
        with pytest.raises(ValueError, match="first must not be negative"):
            select(q, means, seqs, 4, first=first, recent=recent)
    with pytest.raises(ValueError, match="q must have width 64"):
        select(_fake((5, 6, 72)), means, seqs, 4)
    with pytest.raises(ValueError, match="out shape/dtype must match result"):
        select(q, means, seqs, 4, out=_fake((5, 3, 4), torch.int64))


def test_forward_mode_tangents_are_refused():
    from torch.autograd import forward_ad

    seqs = _seqs(2)
    q, k, ids = _fake((5, 6, 64)), _fake((40, 3, 64)), _fake((5, 3, 4), torch.int32)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.zeros(5, 6, 64, dtype=torch.float16),
                                    torch.zeros(5, 6, 64, dtype=torch.float16)).as_subclass(_Cuda)
        with pytest.raises(NotImplementedError, match="q has a forward-mode tangent"):
            fs.flagsparse_block_attention(dual, k, k, ids, seqs)


def _described(**changes):
    c = _lib.FsBlockSeqs()
    c.n_seqs, c.n_tokens, c.n_rows, c.block = 2, 5, 40, 64
    c.q_offsets = c.k_offsets = FAKE
    for name, value in changes.items():
        setattr(c, name, value)
    return c


def test_c_refusals_without_touching_the_gpu():
    lib = _lib.load_library()
    f16, f32, f64 = _lib.FS_F16, _lib.FS_F32, _lib.FS_F64

    def refused(rc, text, code=_lib.FS_E_INVALID):
        assert rc == code and text in lib.fs_last_error().decode(), lib.fs_last_error()

    def attend(c, val=f16, heads=3, group=2, width=64, top=4, q=FAKE, k=FAKE, row=192, scale=0.125, ws=None, need=0):
        return lib.fs_block_attention(val, ctypes.byref(c) if c else None, heads, group, width, top, q, 384, 64, k, 0, row,
                                      64, FAKE, 0, 192, 64, FAKE, 12, 4, scale, FAKE, None, ws, need, None)

    refused(attend(None), "null pointer")
    refused(attend(_described(), val=f64), "value types are")
    refused(attend(_described(n_seqs=-1)), "sizes out of range")
    refused(attend(_described(n_rows=1 << 31)), "sizes out of range")
    refused(attend(_described(n_rows=(1 << 31) - 2047)), "sizes out of range")  # the end of its last block
    refused(attend(_described(block=48)), "blocks are of")
    refused(attend(_described(q_offsets=None)), "without offsets a sequence has one token")
    refused(attend(_described(k_offsets=None)), "null pointer")
    paged = dict(k_offsets=None, pages=FAKE, k_lengths=FAKE, ld_pages=4, pages_per_seq=4, n_pages=9, page_size=16, page_shift=4)
    refused(attend(_described(**{**paged, "page_size": 24})), "power of two")
    refused(attend(_described(**{**paged, "page_shift": 5})), "power of two")
    refused(attend(_described(**{**paged, "k_lengths": None})), "null pointer")
    refused(attend(_described(), heads=0), "heads out of range")
    refused(attend(_described(), group=129), "heads out of range")
    refused(attend(_described(), width=68), "width out of range")
    refused(attend(_described(), val=f32, width=136), "width out of range")
    refused(attend(_described(), top=129), "top out of range")
    refused(attend(_described(), q=None), "bad pointer or stride")
    refused(attend(_described(), k=FAKE + 8), "multiples of 16 bytes")
    refused(attend(_described(), row=196), "multiples of 16 bytes")
    refused(attend(_described(), row=1 << 23), "multiples of 16 bytes")
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        refused(attend(_described(), scale=scale), "scale must be positive")
    many = _described(n_tokens=100000, n_rows=100000)
    need = lib.fs_block_attention_workspace_bytes(f16, ctypes.byref(many), 3, 2, 64, 4)
    assert need > 0
    assert lib.fs_block_attention_workspace_bytes(f16, ctypes.byref(many), 3, 128, 256, 4) == 0  # a token's rows are many
    refused(attend(many, ws=FAKE, need=need - 1), "workspace too small", _lib.FS_E_WORKSPACE)

    most = _described(n_tokens=1 << 27)  # more workgroups of 1024 threads than a launch can have
    refused(attend(most, heads=2, group=12, ws=FAKE, need=1 << 40), "sizes out of range")

    def grad(c, lists=3, top=4, q=FAKE, ws=FAKE, need=1 << 40, dk=FAKE):
        return lib.fs_block_attention_grad(f16, ctypes.byref(c), 3, 2, 64, lists, top, FAKE, q, 384, 64, FAKE, 192, 64,
                                           FAKE, 192, 64, FAKE, 12, 4, 0.125, FAKE, FAKE, FAKE, dk, FAKE, ws, need, None)

    refused(grad(_described(**paged)), "no gradient")
    c = _described()
    refused(lib.fs_block_attention_grad(f16, ctypes.byref(c), 1, 97, 256, 1, 4, FAKE, FAKE, 384, 64, FAKE, 256, 256, FAKE,
                                        256, 256, FAKE, 4, 0, 0.125, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 40, None),
            "heads out of range for this width")
    refused(grad(_described(), lists=2), "lists is 1 or the heads")
    refused(grad(_described(), q=FAKE + 4), "multiples of 16 bytes")
    refused(grad(_described(), dk=None), "bad pointer")
    refused(grad(_described(n_tokens=1 << 28), top=128), "sizes out of range")
    refused(grad(_described(), need=64), "workspace too small", _lib.FS_E_WORKSPACE)

    def select(c, top=4, first=1, recent=1, most=7, means=FAKE):
        return lib.fs_block_select(f16, ctypes.byref(c), 3, 2, 64, FAKE, 384, 64, means, most, 1344, 192, 64, top, first,
                                   recent, FAKE, None)

    refused(select(_described(), top=129), "top, first or recent")
    refused(select(_described(), recent=0), "top, first or recent")
    refused(select(_described(), first=4), "top, first or recent")
    refused(select(_described(), means=None), "bad pointer")
    refused(select(_described(), most=-1), "sizes out of range")
    refused(lib.fs_block_means(f16, ctypes.byref(_described()), 3, 64, None, 0, 192, 64, None, 7, FAKE, 1344, 192, 64, None),
            "bad pointer")
    refused(lib.fs_block_means(f16, ctypes.byref(_described()), 3, 64, FAKE, 0, 192, 64, None, -7, FAKE, 1344, 192, 64, None),
            "sizes out of range")


def test_workspace_sizes():
    lib = _lib.load_library()
    f16 = _lib.FS_F16

    def need(tokens, top, heads=8, block=64):
        c = _described(n_tokens=tokens, n_rows=1 << 20, n_seqs=max(tokens, 1), q_offsets=None, block=block) if tokens < 5000 \
            else _described(n_tokens=tokens, n_rows=1 << 20)
        return lib.fs_block_attention_workspace_bytes(f16, ctypes.byref(c), heads, 4, 128, top)

    assert need(64, 16) == 0  # workgroups enough without splitting
    assert need(1, 128) > 0  # one token with many blocks: several share them
    assert need(0, 16) == 0
    assert need(16384, 16) < 1 << 20  # a word a wave
    c = _described(n_tokens=8192, n_rows=8192, n_seqs=1)
    grads = lib.fs_block_attention_grad_workspace_bytes(f16, ctypes.byref(c), 4, 8, 128, 4, 16)
    assert 8192 * 4 * 16 * 4 * 3 < grads < 1 << 30


@pytest.mark.parametrize("tokens, top, block", [(32768, 16, 64), (131072, 32, 128), (131072, 16, 1024), (1 << 20, 16, 64)])
@pytest.mark.parametrize("lists", [1, 8])
def test_workspace_of_gradients_of_many_tokens(tokens, top, block, lists):
    """What grows with the tokens is some words an entry and a number a row; the sums of
    pieces do not."""
    lib = _lib.load_library()
    heads, group, width = 8, 8, 128
    c = _described(n_tokens=tokens, n_rows=tokens, n_seqs=1, block=block)
    need = lib.fs_block_attention_grad_workspace_bytes(_lib.FS_BF16, ctypes.byref(c), heads, group, width, lists, top)
    entries = tokens * lists * top
    # (a sort in passes has as many words again)
    growing = entries * 4 * 8 + tokens * heads * group * 4 * 2 + 64 * (tokens // block + 2048) * lists
    assert 0 < need < growing + (320 << 20)


@pytest.mark.parametrize("sizes", [dict(n_tokens=1 << 26, n_rows=40), dict(n_tokens=64, n_rows=1 << 29)],
                         ids=["queries", "keys"])
def test_gradients_refuse_launches_that_are_too_large_before_the_first(sizes):
    """More workgroups than a launch can have, of the queries' or of the keys' kernel."""
    lib = _lib.load_library()
    c = _described(**sizes)
    need = lib.fs_block_attention_grad_workspace_bytes(_lib.FS_F16, ctypes.byref(c), 16, 4, 64, 1, 4)
    rc = lib.fs_block_attention_grad(_lib.FS_F16, ctypes.byref(c), 16, 4, 64, 1, 4, FAKE, FAKE, 4096, 64, FAKE, 1024, 64,
                                     FAKE, 1024, 64, FAKE, 4, 0, 0.125, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE,
                                     1 << 50, None)
    assert rc == _lib.FS_E_INVALID and "sizes out of range" in lib.fs_last_error().decode(), lib.fs_last_error()
    assert need == 0


def test_gradients_of_keys_and_values_go_together():
    lib = _lib.load_library()

    def refused(dq, dk, dv):
        c = _described()
        rc = lib.fs_block_attention_grad(_lib.FS_F16, ctypes.byref(c), 3, 2, 64, 3, 4, FAKE, FAKE, 384, 64, FAKE, 192, 64,
                                         FAKE, 192, 64, FAKE, 12, 4, 0.125, FAKE, FAKE, dq, dk, dv, FAKE, 0, None)
        text = lib.fs_last_error().decode()
        return rc == _lib.FS_E_INVALID and "bad pointer" in text, text

    for given in ((FAKE, FAKE, None), (FAKE, None, FAKE), (None, FAKE, None), (None, None, None)):
        assert refused(*given)[0], given
    for given in ((FAKE, FAKE, FAKE), (FAKE, None, None), (None, FAKE, FAKE)):  # (the workspace is)
        bad, text = refused(*given)
        assert not bad and "workspace too small" in text, given
