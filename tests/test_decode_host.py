"""Refusals of the decoding operators and of their C entry points on a host without a GPU."""
import ctypes

import pytest
import torch

from mk_iii_technologies_tsrn_b200 import _lib, ops

P = ctypes.c_void_p(4096)


@pytest.fixture
def lib():
    lib = _lib.load()
    old = lib.tp_set_pointer_checks(0)
    yield lib
    lib.tp_set_pointer_checks(old)


def _cache(**over):
    c = dict(k=P, v=P, pages=4, page_size=16, heads=2, channels=64, k_page=2048, k_slot=128, k_head=64,
             v_page=2048, v_slot=128, v_head=64, table=P, table_row=3, table_cols=3)
    c.update(over)
    return ctypes.byref(_lib.PagedCache(**c))


def test_structure_is_the_headers():
    # two pointers, ten sizes and strides, the table and its two sizes, all of eight bytes
    assert ctypes.sizeof(_lib.PagedCache) == 15 * 8 and _lib.PagedCache.table.offset == 12 * 8


def test_paged_attention_entry_refuses(lib):
    size = lib.tp_paged_attention_workspace_bytes
    need = size(0, 2, 4, 2, 64, 48, 1)
    assert need >= 4 * 2 * 4 * 48 and need % 4 == 0        # the scores at least
    assert size(0, 1, 1, 1, 64, 65536, 0) > 0
    assert size(2, 1, 1, 1, 64, 48, 0) == -1 and size(0, -1, 1, 1, 64, 48, 0) == -1
    assert size(0, 1, 3, 2, 64, 48, 0) == -1 and size(0, 1, 1, 0, 64, 48, 0) == -1
    assert size(0, 0, 4, 2, 64, 48, 1) == 0

    def call(dtype=0, B=2, H=4, lengths=P, q=P, q_sb=256, key=None, value=None, key_sb=128, mass=P,
             mass_sb=96, out=P, ws=P, n=need, **cache):
        return lib.tp_paged_attention(dtype, B, H, _cache(**cache), lengths, q, q_sb, 64, key, key_sb, 64, value,
                                      128, 64, None, None, 0.1, mass, mass_sb, 48, 48, out, ws, n, None)

    assert call(dtype=2) == -4 and call(B=-1) == -1 and call(H=3) == -1 and call(heads=0) == -1
    assert call(channels=0) == -1 and call(channels=257) == -4 and call(page_size=0) == -1
    assert call(pages=-1) == -1 and call(table_cols=-1) == -1 and call(k_slot=-1) == -1
    assert call(table_cols=2 ** 30) == -5 and call(page_size=2 ** 31) == -5
    assert call(q_sb=-1) == -1 and call(key=P) == -1 and call(value=P) == -1
    assert call(key=P, value=P, key_sb=-1) == -1 and call(mass_sb=-1) == -1
    assert call(lengths=None) == -2 and call(q=None) == -2 and call(out=None) == -2
    assert call(k=None) == -2 and call(v=None) == -2 and call(table=None) == -2
    assert call(ws=None) == -7 and call(n=need - 4) == -7 and call(ws=ctypes.c_void_p(4104)) == -3
    assert call(B=2 ** 31) == -5
    assert call(B=0, lengths=None, q=None, out=None, ws=None, k=None) == 0
    assert lib.tp_paged_attention(0, 1, 1, None, P, P, 1, 1, None, 0, 0, None, 0, 0, None, None, 0.1, None, 0, 0,
                                  0, P, None, 0, None) == -2


def test_append_and_evict_entries_refuse(lib):
    def append(dtype=0, B=2, T=3, starts=P, key=P, value=P, st=128, **cache):
        return lib.tp_paged_append(dtype, B, T, _cache(**cache), starts, None, key, 384, st, 64, value, 384, 128,
                                   64, None)

    assert append(dtype=5) == -4 and append(B=-1) == -1 and append(T=-1) == -1 and append(st=-1) == -1
    assert append(starts=None) == -2 and append(key=None) == -2 and append(value=None) == -2
    assert append(T=2 ** 31) == -5 and append(table_row=-1) == -1
    assert append(T=0, starts=None, key=None) == 0 and append(B=0, k=None, table=None) == 0

    def evict(dtype=1, B=2, lengths=P, mass=P, out=P, keep=20, recent=5, kept=P, slots=48, **cache):
        return lib.tp_cache_evict(dtype, B, _cache(**cache), lengths, mass, 96, 48, slots, out, 96, 48, keep,
                                  recent, kept, None)

    assert evict(keep=0) == -1 and evict(recent=-1) == -1 and evict(recent=21) == -1 and evict(slots=-1) == -1
    assert evict(dtype=3) == -4 and evict(B=-1) == -1 and evict(keep=2 ** 31 - 1) == -5
    assert evict(lengths=None) == -2 and evict(mass=None) == -2 and evict(out=None) == -2
    assert evict(kept=None) == -2 and evict(v=None) == -2
    assert evict(B=0, mass=None) == 0 and evict(heads=0, mass=None) == 0


def test_sample_entry_refuses(lib):
    def call(dtype=0, B=2, V=10, logits=P, ld=10, bits=32, uniform=P, token=P):
        return lib.tp_sample_tokens(dtype, B, V, logits, ld, bits, uniform, 1.0, None, 0, None, 1.0, None, 0.0,
                                    None, token, None, None)

    assert call(dtype=2) == -4 and call(B=-1) == -1 and call(V=0) == -1 and call(ld=-1) == -1
    assert call(bits=16) == -1 and call(V=2 ** 19) == -5 and call(B=2 ** 31) == -5
    assert call(logits=None) == -2 and call(uniform=None) == -2 and call(token=None) == -2
    assert call(B=0, logits=None, token=None) == 0


def test_cpu_tensors_and_choices_are_refused():
    q, c = torch.randn(1, 2, 8), torch.randn(3, 4, 2, 8)
    table, n = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    mass, u = torch.zeros(1, 2, 8), torch.rand(1)
    for call in (lambda: ops.paged_attention(q, c, c, table, n),
                 lambda: ops.paged_append(q[:, None], q[:, None], c, c, table, n),
                 lambda: ops.cache_evict(c, c, table, n, mass, 2, 1),
                 lambda: ops.sample_tokens(q[0], u.expand(2).contiguous())):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
    for name, bad in (("temperature", (-0.5, float("nan"))), ("top_k", (-1,)), ("top_p", (0.0, 1.5, float("nan"))),
                      ("min_p", (-0.1, 1.1))):
        for x in bad:
            with pytest.raises(ValueError, match=name):
                ops.sample_tokens(q[0], u, **{name: x})


def test_encoder_layers_without_a_cache_call_their_attention_as_before():
    from mk_iii_technologies_tsrn_b200 import dropin

    class Plain(torch.nn.Module):                 # an attention that knows of no cache
        def forward(self, q, k, v, attn_mask=None, key_padding_mask=None):
            return q, None

    layer = dropin.TropicalEncoderLayer(8, 2, 16, dropout=0.0)
    layer.self_attn, layer.ffn = Plain(), torch.nn.Identity()
    assert layer(torch.randn(1, 3, 8)).shape == (1, 3, 8)
    with pytest.raises(TypeError, match="cache"):
        layer(torch.randn(1, 3, 8), cache=dropin.TropicalKVCache())
