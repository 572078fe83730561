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


# (heads, dim, forks, shared keys, new tokens, us alone, us together): one layer, 32 keys of each fork's own
MEASURED = [
    (8, 128, 2, 256, 1, 9.3, 10.3), (8, 128, 2, 1024, 1, 15.0, 11.8), (8, 128, 4, 1024, 2, 16.1, 13.7),
    (8, 128, 8, 1024, 1, 16.5, 15.5), (8, 128, 16, 256, 1, 10.0, 15.4), (8, 128, 32, 256, 1, 20.3, 15.9),
    (8, 128, 64, 128, 1, 23.8, 17.4), (8, 128, 64, 256, 1, 27.1, 18.4), (8, 128, 64, 8192, 1, 261.4, 31.3),
    (8, 128, 16, 512, 4, 18.5, 22.1), (8, 128, 32, 256, 16, 31.9, 39.3), (8, 128, 64, 1024, 4, 55.2, 34.1),
    (8, 128, 16, 8192, 8, 79.1, 41.8), (8, 128, 16, 8192, 64, 113.4, 172.9),
    (4, 64, 2, 256, 1, 8.2, 10.0), (4, 64, 2, 1024, 1, 13.6, 10.6), (4, 64, 16, 1024, 1, 14.1, 18.7),
    (4, 64, 32, 256, 1, 8.9, 20.4), (4, 64, 64, 256, 1, 10.3, 21.1), (4, 64, 64, 1024, 1, 22.1, 25.3),
    (4, 64, 64, 8192, 1, 79.9, 35.1), (4, 64, 8, 1024, 8, 22.8, 26.9), (4, 64, 16, 8192, 32, 136.9, 161.5),
    (1, 128, 12, 1024, 1, 16.4, 18.9), (1, 128, 64, 2048, 1, 21.6, 27.3)]


@pytest.mark.parametrize("heads,dim,forks,prefix,new,alone,shared", MEASURED)
def test_the_faster_way_is_taken(heads, dim, forks, prefix, new, alone, shared):
    assert together(forks, prefix, new, heads, dim) == (prefix if shared < alone else 0)


def test_the_rule_can_be_moved():
    """The limits are the class's, and an object's own where it has them."""
    c = object.__new__(paged.PagedCache)
    c.page_tokens, c.pool = 16, torch.empty(1, 1, 2, 8, 16, 128, dtype=torch.bfloat16)
    assert c._together([(2, 1)], [1, 1]) == 0
    c.SHARED_KEYS = 16
    assert c._together([(2, 1)], [1, 1]) == 16 and c._together([(1, 0), (1, 0)], [1, 1]) == 0


def test_a_step_without_tokens():
    """Weighs what is not read again like a step of single tokens."""
    assert together(2, 256, [0, 0]) == 0 and together(16, 256, [0] * 16) == 0
    assert together(64, 256, [0] * 64) == 64 * 4
