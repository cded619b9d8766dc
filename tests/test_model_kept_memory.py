"""What the hidden layers of a model hold from the forward to the backward pass, counted in bytes of distinct storages."""
import pytest

from dlrm_amd.model import DLRM, DLRMConfig

BATCH = 96


def model(**options):
    cfg = DLRMConfig(table_rows=[5, 7, 3], dim=128, dense_in=13, bottom=[512, 256, 128], top=[1024, 1024, 512, 256, 1], **options)
    return DLRM(cfg, BATCH, device="cpu", init_tables=False)


def storages(tensors):
    return {t.untyped_storage().data_ptr(): t.untyped_storage().nbytes() for t in tensors}


def outputs(m):
    return m.bot_acts[:-1] + m.top_acts[:-1]


def gradients(m):
    return m.bot_dz + m.top_dz


def kept(m):
    """everything of the hidden layers but the gradients"""
    found = storages(outputs(m))
    for s in (m.bottom, m.top):
        a8 = (s.y8 + s.xhat8) if s.keep8 else []
        found.update(storages([a.codes for a in a8] + [a.exps for a in a8]))
        if s.norm:
            found.update(storages(s.rstd + ([] if s.keep8 else s.z + s.mean)))
    for at in storages(gradients(m)):
        found.pop(at, None)
    return sum(found.values())


@pytest.mark.parametrize("norm", [False, True])
def test_bytes(norm):
    elements = BATCH * (512 + 256 + 1024 + 1024 + 512 + 256)
    statistics = 4 * BATCH * 6 if norm else 0
    tensors = 2 if norm else 1                       # (the outputs, and with norm its inputs or the normalised rows)
    assert kept(model(norm=norm)) == tensors * 4 * elements + 2 * statistics
    assert kept(model(norm=norm, keep8=True)) == tensors * (elements + elements // 32) + statistics


def test_outputs_over_gradients():
    """Widths off every boundary: an output fits into the gradient buffer it lies in, neighbouring layers' do not meet, and the
    gradient buffers are no larger for it."""
    def build(**options):
        cfg = DLRMConfig(table_rows=[5, 7, 3], dim=16, dense_in=13, bottom=[130, 16], top=[33, 301, 257, 61, 1], **options)
        return DLRM(cfg, 3, device="cpu", init_tables=False)
    m, plain = build(keep8=True, norm=True), build(norm=True)
    own = storages(gradients(m))
    assert sorted(own.values()) == sorted(storages(gradients(plain)).values())
    for acts, widths in ((m.bot_acts[:-1], [130]), (m.top_acts[:-1], [33, 301, 257, 61])):
        assert [tuple(a.shape) for a in acts] == [(3, n) for n in widths]
        for a, b in zip(acts, acts[1:]):
            assert a.untyped_storage().data_ptr() != b.untyped_storage().data_ptr()
        for a in acts:
            assert a.untyped_storage().data_ptr() in own and a.stride(1) == 1 and a.stride(0) % 4 == 0
            assert 4 * (a.storage_offset() + 3 * a.stride(0)) <= a.untyped_storage().nbytes()


def test_a_model_without_hidden_layers():
    cfg = DLRMConfig(table_rows=[5], dim=8, dense_in=4, bottom=[8], top=[1], keep8=True, norm=True)
    m = DLRM(cfg, 2, device="cpu", init_tables=False)
    assert outputs(m) == [] and gradients(m) == []
