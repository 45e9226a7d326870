"""Refusals and sizes of the 4-bit KV cache and the 8-bit norm that need no GPU: bad arguments are answered before any device is touched."""
import ctypes as C
import math

import numpy as np
import pytest

import kv4_ref as ref
import x100b

P = 1 << 20   # an aligned address that is never read


def kv(**kw):
    return x100b.Kv4(**dict(dict(pages=P, n_pages=4, page_size=64, n_kv_heads=2, head_dim=128), **kw))


def test_bytes():
    L = x100b.lib()
    # 4.5 bits a value, K and V
    assert L.x100q_kv4_bytes(C.byref(kv())) == 4 * 64 * 2 * 2 * 128 * 9 // 16
    assert L.x100q_kv4_bytes(C.byref(kv(n_pages=1 << 20, head_dim=64, page_size=16))) == (1 << 20) * 16 * 2 * 72
    for bad in (dict(n_pages=0), dict(page_size=48), dict(page_size=256), dict(n_kv_heads=0), dict(n_kv_heads=257), dict(head_dim=96), dict(head_dim=256)):
        assert L.x100q_kv4_bytes(C.byref(kv(**bad))) == 0
    assert L.x100q_kv4_bytes(None) == 0


APPEND = dict(dtype=0, n_tokens=3, n_heads=4, q=P, k=P, v=P, q_out=P, q_stride=512, k_stride=256, v_stride=256, q_out_stride=512, q_norm=0, k_norm=0,
              eps=1e-6, rope=P, rope_len=8, pos=P, seq=P, page_table=P, table_stride=2, n_seqs=2)


@pytest.mark.parametrize("bad", [dict(n_tokens=-1), dict(k=0), dict(v=0), dict(pos=0), dict(page_table=0), dict(table_stride=0), dict(n_seqs=0), dict(k=P + 4),
                                 dict(k_stride=255), dict(v_stride=258), dict(q_stride=508), dict(q_out=0), dict(q=P + 8), dict(n_heads=0), dict(rope_len=0),
                                 dict(seq=0), dict(q_norm=P, eps=-1.0), dict(k_norm=P, eps=math.nan), dict(rope=P + 4)])
def test_append_refusals(bad):
    a = x100b.Kv4AppendArgs(**dict(APPEND, **bad))
    assert x100b.lib().x100q_kv4_append_dev(C.byref(kv()), C.byref(a), None) == x100b.X100_E_ARG
    assert x100b.last_error() == x100b.X100_E_ARG


ATTN = dict(dtype=1, n_heads=4, q=P, out=P, q_stride=512, out_stride=512, q_start=P, n_tokens=3, max_q=2, kv_len=P, page_table=P, table_stride=2, n_seqs=2,
            scale=0.1, work=P, work_bytes=1 << 30)


@pytest.mark.parametrize("bad", [dict(n_heads=3), dict(n_heads=0), dict(q=0), dict(out=P + 2), dict(q_stride=511), dict(out_stride=384), dict(q_start=0),
                                 dict(n_tokens=-1), dict(max_q=0), dict(kv_len=0), dict(page_table=0), dict(table_stride=0), dict(n_seqs=0), dict(scale=0.0),
                                 dict(scale=math.inf), dict(scale=math.nan), dict(work=0), dict(work=P + 4)])
def test_attention_refusals(bad):
    a = x100b.Kv4AttnArgs(**dict(ATTN, **bad))
    assert x100b.lib().x100q_kv4_attn_dev(C.byref(kv()), C.byref(a), None) == x100b.X100_E_ARG


def test_other_codes():
    L = x100b.lib()
    assert L.x100q_kv4_attn_dev(C.byref(kv()), C.byref(x100b.Kv4AttnArgs(**dict(ATTN, dtype=8))), None) == x100b.X100_E_UNSUPPORTED
    assert L.x100q_kv4_append_dev(C.byref(kv()), C.byref(x100b.Kv4AppendArgs(**dict(APPEND, dtype=2))), None) == x100b.X100_E_UNSUPPORTED
    need = L.x100q_kv4_attn_work(C.byref(kv()), 3, 4, 2)
    assert need > 0 and L.x100q_kv4_attn_work(C.byref(kv()), 3, 3, 2) == 0
    assert L.x100q_kv4_attn_dev(C.byref(kv()), C.byref(x100b.Kv4AttnArgs(**dict(ATTN, work_bytes=need - 1))), None) == x100b.X100_E_TOO_LARGE
    for fn, base in ((L.x100q_kv4_append_dev, x100b.Kv4AppendArgs(**dict(APPEND, n_tokens=0))), (L.x100q_kv4_attn_dev, x100b.Kv4AttnArgs(**dict(ATTN, n_tokens=0)))):
        assert fn(C.byref(kv()), C.byref(base), None) == x100b.X100_OK        # nothing to do
        assert fn(C.byref(kv(page_size=17)), C.byref(base), None) == x100b.X100_E_ARG
        assert fn(C.byref(kv()), None, None) == x100b.X100_E_ARG
    assert L.x100q_kv4_append_dev(C.byref(kv(pages=P + 8)), C.byref(x100b.Kv4AppendArgs(**APPEND)), None) == x100b.X100_E_ARG
    assert L.x100q_kv4_read_dev(C.byref(kv()), P, None, 3, P, 2, 2, P, P, None) == x100b.X100_E_ARG      # more tokens than sequences
    assert L.x100q_kv4_read_dev(C.byref(kv()), P, P, 3, P, 2, 2, P + 2, P, None) == x100b.X100_E_ARG
    assert L.x100q_kv4_read_dev(C.byref(kv()), P, P, 0, P, 2, 2, P, P, None) == x100b.X100_OK
    assert L.x100q_rope_table_dev(P, 4, 7, 1e4, None) == x100b.X100_E_ARG and L.x100q_rope_table_dev(P, 4, 8, 0.0, None) == x100b.X100_E_ARG


NORM = dict(dtype=0, rows=4, d=256, group=0, x=P, residual=P, residual_out=P, ldx=256, ldr=256, ldo=256, ldq=256, w=P, eps=1e-6, q=P, scales=P)


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(d=0), dict(x=0), dict(w=0), dict(q=0), dict(scales=0), dict(eps=0.0), dict(eps=math.nan), dict(ldx=255),
                                 dict(ldq=255), dict(ldr=255), dict(ldo=255), dict(group=16), dict(group=96), dict(group=-32), dict(d=240, group=128),
                                 dict(x=P + 2), dict(residual=0)])
def test_norm_refusals(bad):
    a = x100b.NormQ8Args(**dict(NORM, **bad))
    assert x100b.lib().x100q_add_rmsnorm_q8_dev(C.byref(a), None) == x100b.X100_E_ARG


def test_norm_other_codes():
    L = x100b.lib()
    assert L.x100q_add_rmsnorm_q8_dev(C.byref(x100b.NormQ8Args(**dict(NORM, dtype=2))), None) == x100b.X100_E_UNSUPPORTED
    assert L.x100q_add_rmsnorm_q8_dev(C.byref(x100b.NormQ8Args(**dict(NORM, rows=0))), None) == x100b.X100_OK
    assert L.x100q_add_rmsnorm_q8_dev(None, None) == x100b.X100_E_ARG


def test_struct_layouts_follow_the_header():
    """The ctypes structures list the header's fields in order."""
    import re
    src = re.sub(r"/\*.*?\*/", "", open(x100b.HEADERS[1]).read(), flags=re.S)
    for name, st in (("x100q_kv4", x100b.Kv4), ("x100q_kv4_append_args", x100b.Kv4AppendArgs), ("x100q_kv4_attn_args", x100b.Kv4AttnArgs),
                     ("x100q_norm_q8_args", x100b.NormQ8Args)):
        body = re.search(r"typedef struct \{([^}]*)\} " + name + ";", src).group(1)
        fields = [re.sub(r"^.*[\s*]", "", f.strip()) for line in body.split(";") for f in line.split(",") if f.strip()]
        assert fields == [f for f, _ in st._fields_]


def test_reference_scales_make_fp16_values():
    """d * (code - 8) is an fp16 value for every scale of 8 significand bits, the smallest and largest among them."""
    d = ref.scale16(np.concatenate([np.float32(2.0) ** np.arange(-30, 14), np.random.default_rng(0).normal(size=4000) * 10.0 ** np.arange(-4, 4).repeat(500)]))
    v = d.astype(np.float64)[:, None] * np.arange(-8, 8)
    assert np.array_equal(v.astype(np.float16).astype(np.float64), v)


MODEL = dict(n_layers=1, d=512, n_heads=16, n_kv_heads=2, head_dim=128, vocab=64, n_exp=8, n_act=2, moe_ffn=256, attn_qtype=x100b.Q8_0,
             expert_qtype=x100b.Q8_0, lm_qtype=x100b.Q8_0, ctx=64, max_batch=2, expert_lo=0, expert_hi=8, rope_base=1e6, eps=1e-6)


@pytest.mark.parametrize("pool", [dict(n_kv_heads=4), dict(head_dim=64), dict(pages=0), dict(pages=P + 8), dict(page_size=8), dict(n_pages=0)])
def test_model_refuses_another_pool(pool):
    L, cfg = x100b.lib(), x100b.ModelCfg(**MODEL)
    assert L.x100q_model_create_kv4(C.byref(cfg), C.byref(kv(**pool)), P, 2) is None
    assert x100b.last_error() == x100b.X100_E_ARG


def test_model_refuses_no_pool_or_table():
    L, cfg = x100b.lib(), x100b.ModelCfg(**MODEL)
    for args in ((None, P, 2), (C.byref(kv()), None, 2), (C.byref(kv()), P, 0)):
        assert L.x100q_model_create_kv4(C.byref(cfg), *args) is None and x100b.last_error() == x100b.X100_E_ARG
    assert L.x100q_model_load_gguf_kv4(None, C.byref(cfg), C.byref(kv()), P, 2) is None and x100b.last_error() == x100b.X100_E_ARG


def test_scratch_follows_the_rows_a_sequence_can_have():
    """256 rows (tokens times query heads per kv head) need the prompt kernel's scratch, fewer the other's; neither depends on lengths."""
    L, p = x100b.lib(), C.byref(kv())
    few, many = L.x100q_kv4_attn_work(p, 1, 2, 1), L.x100q_kv4_attn_work(p, 4096, 32, 1)
    assert 0 < few < many
    assert L.x100q_kv4_attn_work(p, 255, 2, 3) == few and L.x100q_kv4_attn_work(p, 256, 2, 3) == many
    assert L.x100q_kv4_attn_work(p, 31, 16, 1) == few and L.x100q_kv4_attn_work(p, 32, 16, 1) == many


@pytest.mark.parametrize("big", [dict(n_seqs=4096, max_q=1 << 19), dict(n_seqs=64, max_q=1 << 19, table_stride=1 << 20), dict(n_seqs=1, max_q=1 << 20), dict(n_seqs=65537)])
def test_calls_past_the_work_list_are_refused(big):
    a = x100b.Kv4AttnArgs(**dict(ATTN, n_tokens=1 << 20, work_bytes=1 << 40, **big))
    assert x100b.lib().x100q_kv4_attn_dev(C.byref(kv()), C.byref(a), None) == x100b.X100_E_TOO_LARGE


@pytest.mark.parametrize("pack,args", [(x100b._APPEND, x100b.Kv4AppendArgs), (x100b._ATTN, x100b.Kv4AttnArgs), (x100b._NORM, x100b.NormQ8Args)])
def test_packed_arguments_are_the_structs(pack, args):
    values = [1 + 3 * i for i in range(len(args._fields_))]
    raw = pack(*values)
    assert len(raw) == C.sizeof(args)
    assert [getattr(args.from_buffer_copy(raw), name) for name, _ in args._fields_] == values
