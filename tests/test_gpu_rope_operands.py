"""qk_rope's copies of operands live until the launch that reads them."""
import pytest
import torch

from gpu_util import normal

pytestmark = pytest.mark.gpu


def test_copies_outlive_the_launch(pkg, dev, monkeypatch):
    """Every operand in a layout that is copied first: none of the copies may be
    memory that another thread of the same stream could be given before the launch."""
    T, H, d = 5, 4, 64
    freq, axis = pkg.rope_frequencies(d, sections=(20, 12), device=dev)
    plain = (normal((T, H, d), 1).to(dev), normal((T, 2, d), 2).to(dev), torch.arange(2 * T, device=dev).view(2, T), freq)
    weights = dict(q_weight=normal((d,), 3).to(dev), k_weight=normal((d,), 4).to(dev))
    want = pkg.qk_rope(*plain, axis=axis, **weights)
    spread = lambda t: t.repeat_interleave(2, -1)[..., ::2]  # noqa: E731
    real, seen = pkg.load_library(), []

    class Library:
        def __getattr__(self, name):
            return getattr(real, name)

        def hxmi_qk_rope(self, *args):
            read = {args[i] for i in (1, 2, 5, 7, 8, 9, 10)}
            sizes = [(t.numel() * t.element_size()) for t in (*plain, axis, *weights.values())]
            again = [torch.empty(n, dtype=torch.uint8, device=dev) for n in sizes for _ in range(3)]
            seen.append(not read & {t.data_ptr() for t in again})
            return real.hxmi_qk_rope(*args) if seen[-1] else 0

    monkeypatch.setattr(pkg.hxmi, "load_library", lambda: Library())
    got = pkg.qk_rope(*map(spread, plain), axis=spread(axis), **{n: spread(w) for n, w in weights.items()})
    assert seen == [True]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
