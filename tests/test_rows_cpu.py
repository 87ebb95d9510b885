"""Row operators without a GPU: public names, checks made before any launch, and
the C entry points' refusals and workspace sizes."""

import inspect

import pytest
import torch

import flagsparse_amd as fs
from flagsparse_amd import _lib

NAMES = {
    "flagsparse_embedding", "flagsparse_embedding_grad", "PreparedExpertRoute", "prepare_expert_route",
    "flagsparse_expert_dispatch", "flagsparse_expert_dispatch_grad", "flagsparse_expert_combine",
    "flagsparse_expert_combine_grad", "flagsparse_expert_product", "flagsparse_expert_product_grad",
}
FAKE = 4096  # an address that no refused call reads


def test_public_names():
    assert NAMES <= set(fs.__all__) and NAMES <= set(dir(fs))
    for name in NAMES:
        assert inspect.getdoc(getattr(fs, name))


def test_cpu_tensors_are_refused():
    ids, table = torch.tensor([0, 1]), torch.ones(3, 4)
    with pytest.raises(ValueError, match="table and tokens must be CUDA tensors"):
        fs.flagsparse_embedding(table, ids)
    with pytest.raises(ValueError, match="grad and tokens must be CUDA tensors"):
        fs.flagsparse_embedding_grad(table[:2], ids, 3)
    with pytest.raises(ValueError, match="experts must be a CUDA tensor"):
        fs.prepare_expert_route(ids[:, None], 2)
    for call in (fs.flagsparse_expert_dispatch, fs.flagsparse_expert_dispatch_grad, fs.flagsparse_expert_combine):
        with pytest.raises(TypeError, match="route must be a PreparedExpertRoute"):
            call(table, None)
    with pytest.raises(TypeError, match="table and tokens must be torch.Tensor"):
        fs.flagsparse_embedding([[1.0]], ids)


def test_c_refusals_without_touching_the_gpu():
    lib = _lib.load_library()
    f32, f64, c64, i64 = _lib.FS_F32, _lib.FS_F64, _lib.FS_C64, _lib.FS_I64

    def refused(rc, text, code=_lib.FS_E_INVALID):
        assert rc == code and text in lib.fs_last_error().decode(), lib.fs_last_error()

    refused(lib.fs_embedding(c64, i64, 1, 4, 8, FAKE, 8, FAKE, 1.0, FAKE, None), "bad value type")
    refused(lib.fs_embedding(f32, 7, 1, 4, 8, FAKE, 8, FAKE, 1.0, FAKE, None), "bad type code")
    refused(lib.fs_embedding(f32, i64, -1, 4, 8, FAKE, 8, FAKE, 1.0, FAKE, None), "sizes out of range")
    refused(lib.fs_embedding(f32, i64, 1, 4, 8, None, 8, FAKE, 1.0, FAKE, None), "bad pointer")
    refused(lib.fs_embedding_grad(f32, _lib.FS_F16, i64, 1, 4, 8, FAKE, 8, FAKE, 1.0, -1, FAKE, FAKE, 1 << 20, None),
            "gradient's type or float32")
    refused(lib.fs_embedding_grad(f32, f32, i64, 1, 4, 8, FAKE, 8, FAKE, 1.0, -1, FAKE, FAKE, 8, None),
            "workspace too small", _lib.FS_E_WORKSPACE)
    refused(lib.fs_expert_route(i64, 8, 0, FAKE, FAKE, FAKE, FAKE, None, 0, None), "n_experts out of range")
    refused(lib.fs_expert_route(i64, 8, 1024, FAKE, FAKE, FAKE, FAKE, None, 0, None), "n_experts out of range")
    refused(lib.fs_expert_route(i64, 1 << 31, 8, FAKE, FAKE, FAKE, FAKE, None, 0, None), "slots out of range")
    refused(lib.fs_expert_route(i64, 5000, 8, FAKE, FAKE, FAKE, FAKE, None, 0, None), "workspace too small",
            _lib.FS_E_WORKSPACE)
    refused(lib.fs_expert_dispatch(f32, 1 << 30, 2, 8, 4, FAKE, 8, FAKE, FAKE, FAKE, None), "sizes out of range")
    refused(lib.fs_expert_combine(f32, 4, 0, 8, 4, FAKE, 8, FAKE, FAKE, None, FAKE, None), "sizes out of range")
    refused(lib.fs_expert_combine(f32, 4, 2, 8, 4, FAKE, -8, FAKE, FAKE, None, FAKE, None), "bad pointer or stride")
    refused(lib.fs_expert_combine_grad(f32, 4, 2, 8, 4, FAKE, 8, FAKE, 8, FAKE, FAKE, None, FAKE, FAKE, None),
            "bad pointer or stride")
    refused(lib.fs_expert_product(f64, 0, 8, 2, 16, 16, FAKE, 16, FAKE, FAKE, FAKE, None, 0, None), "value types are")
    refused(lib.fs_expert_product(f32, 2, 8, 2, 16, 16, FAKE, 16, FAKE, FAKE, FAKE, None, 0, None), "sizes out of range")
    refused(lib.fs_expert_product(f32, 0, 8, 2, 16, 16, None, 16, FAKE, FAKE, FAKE, None, 0, None), "bad pointer")
    refused(lib.fs_expert_product_grad_matrices(f32, 0, 8, 2, 16, 16, FAKE, 16, None, 16, FAKE, FAKE, None, 0, None),
            "bad pointer")
    # no workspace where tiles of the last round may be shared
    args = (_lib.FS_BF16, 0, 8192, 8, 4096, 4096)
    assert lib.fs_expert_product_workspace_bytes(*args) > 0
    refused(lib.fs_expert_product(*args, FAKE, 4096, FAKE, FAKE, FAKE, None, 0, None), "workspace too small",
            _lib.FS_E_WORKSPACE)


def test_workspace_sizes():
    lib = _lib.load_library()
    assert lib.fs_expert_route_workspace_bytes(4096, 64) == 0  # one workgroup sorts them
    assert lib.fs_expert_route_workspace_bytes(5000, 64) > 0
    assert lib.fs_expert_route_workspace_bytes(0, 64) == 0
    assert lib.fs_embedding_grad_workspace_bytes(_lib.FS_F32, 0, 100, 8) == 0
    small = lib.fs_embedding_grad_workspace_bytes(_lib.FS_F32, 64, 100, 8)
    assert small >= 2 * 64 * 4
    # sums of 64 positions, two a chunk
    assert lib.fs_embedding_grad_workspace_bytes(_lib.FS_F32, 6400, 100, 8) >= 2 * 100 * 8 * 4
    assert (lib.fs_embedding_grad_workspace_bytes(_lib.FS_F64, 6400, 100, 8)
            > lib.fs_embedding_grad_workspace_bytes(_lib.FS_F32, 6400, 100, 8))
    assert lib.fs_expert_product_workspace_bytes(_lib.FS_F32, 0, 8192, 8, 4096, 4096) == 0
    assert lib.fs_expert_product_workspace_bytes(_lib.FS_BF16, 0, 16, 8, 4096, 4096) == 0
