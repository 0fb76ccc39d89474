"""The attention over pages, as compiled: at each of its barriers no LDS access of the wave is in flight (its wide tiles refill a
buffer behind a barrier that orders nothing else)."""
from test_kernel_waits import _assembly, _functions, _pending_at_barriers


def test_no_lds_access_crosses_a_barrier(tmp_path):
    seen = 0
    for name, body in _functions(_assembly("page_attention", tmp_path)):
        if "k_page_attn" not in name or "join" in name:
            continue
        seen += 1
        barriers = _pending_at_barriers(body)
        assert len(barriers) >= 4, name
        assert all(n == 0 for n in barriers.values()), (name, barriers)
    assert seen == 2


def test_none_crosses_a_barrier_of_few_rows(tmp_path):
    seen = 0
    for name, body in _functions(_assembly("page_attention", tmp_path)):
        if "k_page_few" not in name:
            continue
        seen += 1
        barriers = _pending_at_barriers(body)
        assert len(barriers) >= 3, name
        assert all(n == 0 for n in barriers.values()), (name, barriers)
    assert seen == 4
