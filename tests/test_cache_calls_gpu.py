"""What a call of the cache and attention operators leaves behind for autograd: its knowledge of what was overwritten."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _ops(built_libs):
    import distserve_b200

    distserve_b200.load_ops()


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def calls():
    """Each operator: a function of its tensors, which it is given, and the names of those that it writes."""
    rows = lambda n, h: torch.randn(n, h, 64, device="cuda").half()  # noqa: E731
    pool = lambda: torch.zeros(4, 1, 2, 16, 64, dtype=torch.float16, device="cuda")  # noqa: E731
    table, lens, starts = ints(0)[None], ints(3), ints(0, 3)
    new = dict(k=rows(3, 2), v=rows(3, 2), k_cache=pool(), v_cache=pool())
    yield ("k_cache", "v_cache"), new, lambda t: torch.ops.kv_cache_ops.write(t["k"], t["v"], t["k_cache"], t["v_cache"], 0, table, lens, starts)
    new = dict(k=rows(3, 2), v=rows(3, 2), k_cache=pool(), v_cache=pool())
    yield ("k", "v"), new, lambda t: torch.ops.kv_cache_ops.read(t["k_cache"], t["v_cache"], 0, table, starts, t["k"], t["v"])
    new = dict(q=rows(3, 4), out=rows(3, 4), k_cache=pool(), v_cache=pool())
    yield ("out",), new, lambda t: torch.ops.kv_attention_ops.paged(t["q"], t["k_cache"], t["v_cache"], 0, table, lens, starts, 3, 0.1, t["out"])
    new = dict(q=rows(3, 4), k=rows(3, 2), v=rows(3, 2), out=rows(3, 4))
    yield ("out",), new, lambda t: torch.ops.kv_attention_ops.prompt(t["q"], t["k"], t["v"], starts, 3, 0.1, t["out"])


def test_what_is_written_counts_as_written():
    for written, tensors, call in calls():
        before = {name: t._version for name, t in tensors.items()}
        call(tensors)
        for name, t in tensors.items():
            assert (t._version > before[name]) == (name in written), name
        # a tensor that autograd has saved and that a call then overwrites: the backward pass says so
        x = torch.ones((), device="cuda", dtype=torch.float16, requires_grad=True)
        y = (x * tensors[written[0]]).sum()
        with torch.no_grad():
            call(tensors)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    torch.cuda.synchronize()


def test_tensors_made_in_inference_mode():
    with torch.inference_mode():
        made = [(tensors, call) for _, tensors, call in calls()]
        for tensors, call in made:
            call(tensors)
    for tensors, call in made:                     # and used outside it
        call(tensors)
    torch.cuda.synchronize()
