"""HbmExpertStore.put_expert and the layer's table, with a store in host memory (no GPU needed: the quantisation is
left out)."""
import pytest
import torch

from home_seek_amd import expert_store, ops

D, I = 256, 128


@pytest.fixture()
def store(monkeypatch):
    monkeypatch.setattr(ops, "fp4_quant", lambda w, out: out)
    return expert_store.HbmExpertStore(1, 4, D, I, "cpu", with_shared=False)


def weights():
    return torch.zeros(I, D), torch.zeros(I, D), torch.zeros(D, I)


def test_an_absent_expert_gets_its_row_of_the_table(store):
    want = store.table(0).clone()
    store.mark_absent(0, 2)
    table = store.table(0)
    assert (table[2] == 0).all()
    store.put_expert(0, 2, *weights())
    assert store.has_expert(0, 2) and store.table(0) is table and torch.equal(table, want)


def test_an_expert_whose_row_was_not_written_stays_absent(store):
    """A table that cannot be written (a copy from host memory inside a graph capture, say): the next call tries again."""
    want = store.table(0).clone()
    store.mark_absent(0, 2)
    table = store.table(0)

    class Refuses:
        def __getitem__(self, eid):
            raise RuntimeError("not now")

    store._tables[0] = Refuses()
    with pytest.raises(RuntimeError, match="not now"):
        store.put_expert(0, 2, *weights())
    assert not store.has_expert(0, 2)
    store._tables[0] = table
    store.put_expert(0, 2, *weights())
    assert store.has_expert(0, 2) and torch.equal(store.table(0), want)
