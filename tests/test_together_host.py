"""Which steps' forks attend to their shared keys together, without a GPU."""
import pytest

torch = pytest.importorskip("torch")

from llm_accelerator_b200 import paged  # noqa: E402


def together(forks, prefix, counts, heads=8, dim=128, page=64, strangers=0):
    c = object.__new__(paged.PagedCache)
    c.page_tokens, c.pool = page, torch.empty(1, 1, 2, heads, page, dim, dtype=torch.bfloat16)
    counts = [counts] * (forks + strangers) if isinstance(counts, int) else counts
    return c._together([(forks, prefix // page)] + [(1, 0)] * strangers, counts)


@pytest.mark.parametrize("forks,prefix", [(2, 1024), (2, 8192), (16, 8192), (64, 1024), (64, 65536)])
def test_long_chunks_attend_alone(forks, prefix):
    """Chunks that fill tiles of rows by themselves were up to three times slower together."""
    for new in (32, 64, 256, 4096):
        assert together(forks, prefix, new) == 0
    assert together(forks, prefix, [1] * forks) == prefix
    assert together(forks, prefix, [1] * (forks - 1) + [512]) == 0
    assert together(forks, prefix, [1] * forks + [300], strangers=1) == 0
