"""CPU: a workspace sized for the largest call serves every smaller one: sizes never fall as tokens, rows or elements grow."""
import pytest

from ddgani_amd import _lib


def rising(size, points):
    last = 0
    for n in sorted(points):
        got = size(n)
        assert got >= last, (n, got, last)
        last = got


@pytest.mark.parametrize("D", [1, 7, 256, 2048])
def test_embedding_grad(D):
    ends = [1024, 65536, 135041, 1 << 20, 1 << 22, (1 << 31) - 1]
    rising(lambda n: _lib.lib().ddg_embedding_grad_workspace_bytes(n, D), {m + d for m in ends for d in (-2, -1, 0)} | set(range(0, 3000000, 9973)))


@pytest.mark.parametrize("name", ["ddg_fp8_linear_workspace_bytes", "ddg_fp8_linear_grads_workspace_bytes"])
@pytest.mark.parametrize("out,inn", [(4096, 4096), (64, 64), (1000, 8192), (352, 176), (5000, 2048), (1, 100000), (8192, 1)])
def test_fp8(name, out, inn):
    points = set(range(1, 2100)) | {128 * t + d for t in range(16, 900) for d in (0, 1)} | {1 << 17, 200000, 1 << 20, (1 << 24) - 200}
    rising(lambda rows: getattr(_lib.lib(), name)(rows, out, inn), points)


def test_adamw():
    def size(numel, more=0):
        t = (_lib.AdamwTensor * (1 + more))(*[_lib.AdamwTensor(None, None, n, 0, 0.0, 0, 0, 0) for n in [numel] + [700] * more])
        return _lib.lib().ddg_adamw_workspace_bytes(t, 1 + more)
    rising(size, set(range(1, 6000000, 30011)) | {1 << 20, (1 << 20) + 1})
    rising(lambda more: size(1000000, more), range(200))
