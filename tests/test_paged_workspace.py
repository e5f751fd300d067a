"""What aq_paged_attention_workspace promises, on the host alone: the bytes for a batch's largest bounds serve every batch
within them. What a call itself needs is read from its refusal of a workspace of no bytes, which comes before anything
touches a device."""
import random
import re

import pytest

import aqueduct as aq
from test_paged_refusals import FAKE, FakeCtx, good_batch, good_kv, rows


@pytest.fixture()
def ctx():
    return FakeCtx()


def batch(n_seq, n_rows, max_rows, max_len, cols=1 << 12):
    return good_batch(n_seq=n_seq, n_rows=n_rows, max_rows=max_rows, max_pages=cols, max_len=max_len)


def needs(ctx, kv, b, heads):
    """Bytes that the calls with rows of either type need."""
    out = []
    for t in {aq.F32, kv.type}:
        x = rows(t=t, heads=heads, hd=kv.head_dim)
        with pytest.raises(aq.AqError) as e:
            aq.paged_attention(ctx, kv, b, heads, x, x, 0.1, workspace=FAKE, workspace_bytes=0)
        out.append(int(re.search(r"(\d+) needed", str(e.value)).group(1)))
    return out


@pytest.mark.parametrize("hd,heads,big,small", [
    (256, 8, (1, 11, 9, 16), (1, 11, 2, 3)), (256, 1, (2, 58, 23, 6), (2, 58, 7, 1)),
    (128, 8, (1, 11, 11, 2), (1, 11, 2, 2)), (64, 4, (1, 90, 7, 555), (1, 90, 1, 523))])
def test_fewer_rows_a_sequence(ctx, hd, heads, big, small):
    kv = good_kv(n_head_kv=1, head_dim=hd, type=aq.F32)
    assert max(needs(ctx, kv, batch(*small), heads)) <= aq.paged_attention_workspace(ctx, kv, batch(*big), heads)


def test_every_bound_for_itself(ctx):
    """Sequences, rows, rows of a sequence, positions and table columns drawn one by one within the larger bounds."""
    rng = random.Random(5)

    def log(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    for _ in range(6000):
        n_kv = rng.choice([1, 2, 4, 8])
        kv = good_kv(n_head_kv=n_kv, head_dim=rng.choice([64, 80, 128, 192, 256]), type=rng.choice([aq.F32, aq.F16, aq.BF16]))
        heads = n_kv * rng.choice([1, 2, 4, 6, 12])
        big = [log(1, 3000), log(1, 30000), log(1, 3000), log(1, 60000), log(1, 4096)]
        small = [rng.choice([b, log(1, b)]) for b in big]
        have = aq.paged_attention_workspace(ctx, kv, batch(*big), heads)
        what = (big, small, kv.type, kv.head_dim, n_kv, heads)
        assert aq.paged_attention_workspace(ctx, kv, batch(*small), heads) <= have, what
        for b in (big, small):
            assert max(needs(ctx, kv, batch(*b), heads)) <= have, what
