"""What the cache and attention operators refuse before they look for a device: calls that autograd would have to follow, and
workspaces that do not fit."""
import pytest
import torch
from torch.autograd import forward_ad


@pytest.fixture(scope="module", autouse=True)
def _ops(built_libs):
    import distserve_b200

    distserve_b200.load_ops()


def calls(change):
    """Each operator with one of its tensors, each in turn, replaced by what `change` makes of it."""
    ints = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    table, lens, starts = ints(0)[None], ints(3), ints(0, 3)
    cache, attention = torch.ops.kv_cache_ops, torch.ops.kv_attention_ops
    forms = [
        (4, lambda a, b, kc, vc: cache.write(a, b, kc, vc, 0, table, lens, starts)),
        (4, lambda a, b, kc, vc: cache.read(kc, vc, 0, table, starts, a, b)),
        (4, lambda a, b, kc, vc: attention.paged(a, kc, vc, 0, table, lens, starts, 3, 0.1, b)),
        (4, lambda a, b, c, d: attention.prompt(a, b, c, starts, 3, 0.1, d)),
    ]
    for which, (count, form) in enumerate(forms):
        for i in range(count):
            tensors = [torch.randn(3, 2, 64).half() for _ in range(4)]
            if which < 3:
                tensors[2:] = [torch.randn(4, 1, 2, 16, 64).half() for _ in range(2)]
            tensors[i] = change(tensors[i])
            yield lambda f=form, t=tensors: f(*t)


def test_forward_mode_tangents_are_refused():
    """They do not show in requires_grad, and count under no_grad too."""
    with forward_ad.dual_level():
        for call in calls(lambda t: forward_ad.make_dual(t, torch.ones_like(t))):
            with pytest.raises(RuntimeError, match="has no gradient, and an argument carries a forward-mode tangent"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="has no gradient, and"):
                call()


def test_leaves_that_require_a_gradient_are_refused():
    for call in calls(lambda t: t.requires_grad_()):
        with pytest.raises(RuntimeError, match="has no gradient: call it under torch.no_grad"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA tensor"):       # then only the device is missing
            call()


@pytest.mark.parametrize("elem_size", [1, 2])
@pytest.mark.parametrize("num_seqs,max_rows", [(1, 1), (3, 4), (2, 300)])
def test_a_workspace_that_does_not_fit_is_refused(built_libs, num_seqs, max_rows, elem_size):
    """Partial results go there, so it is what keeps them in bounds: too small, absent or misaligned never reaches a launch."""
    from distserve_b200 import capi

    shape = capi.PoolShape.of(num_blocks=4096, num_layers=2, num_heads=2, block_size=16, head_dim=64 + (4 if elem_size == 1 else 0), elem_size=elem_size)
    rows = capi.Rows(0x1000, 8, 512, 64)
    batch = capi.Batch(num_seqs, num_seqs * max_rows, max_rows, 0x9000, 0xA000, 0xB000, 1024, 1024)
    need = capi.paged_attention_workspace(shape, 8, batch)
    assert need > 0 and need == capi.paged_attention_workspace(shape, 8, batch)

    def call(workspace, size):
        capi.paged_attention(rows, rows, 0, 0x100000, 0x200000, shape, 1, batch, 0.125, workspace, size)

    for workspace, size in ((0x40000, need - 1), (0x40000, 0), (0x40000, -1), (0, need), (0x40008, need), (0x40001, 2 * need)):
        with pytest.raises(capi.KvmigError, match=f"needs a workspace of {need} bytes") as e:
            call(workspace, size)
        assert e.value.code == capi.EINVAL
    if not torch.cuda.is_available():
        with pytest.raises(capi.KvmigError, match="cudaGetDevice"):         # enough of it: then only the device is missing
            call(0x40000, need)
