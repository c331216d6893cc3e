"""The binding's cache calls refuse tensors of types that the library would read past their end or as other numbers,
before anything is called (no GPU)."""
import pytest


def make():
    import mako_attn
    import torch
    h, x = torch.zeros(4096, dtype=torch.float16), torch.zeros(512)
    n, f = torch.zeros(4, dtype=torch.int32), torch.zeros(64, dtype=torch.float64)
    c = object.__new__(mako_attn.Context)  # no device here
    c._h, c.device = None, 0
    common = dict(k=h, v=h, kv_len=n, kv_heads=1, dim=128, k_stride=8)
    calls = dict(
        cache_append=dict(common, x=x, ld=512, q_col0=0, q_stride=128, k_col0=256, v_col0=384, batch=1, n_tok=1, n_new=n,
                          pos=n, heads=2, rot=128, layout=1, freq=f, amplitude=1.0, wq=x, wk=x, eps=1e-6, q=h, weight=x),
        attention_tree=dict(common, q=h, o=x, batch=1, n_tok=2, n_new=n, max_kv_len=6, heads=2, mask=n),
        attention_decode_weights=dict(common, q=h, o=x, weight=x, max_kv_len=8, heads=2),
        cache_evict=dict(common, weight=x, max_kv_len=8, sinks=1, recent=1, budget=4, k_out=h, v_out=h, weight_out=x,
                         out_stride=4, kept=n, new_len=n))
    return c, calls


@pytest.mark.parametrize("name", ["cache_append", "attention_tree", "attention_decode_weights", "cache_evict"])
def test_other_types_are_refused(name, monkeypatch):
    import mako_attn
    import torch
    c, calls = make()
    ok = calls[name]
    reached = []
    mako_attn._load_types()
    monkeypatch.setattr(mako_attn, "_raw_stream", lambda device: 0)
    monkeypatch.setattr(mako_attn, "_check", reached.append)
    getattr(c, name)(**ok)  # the library refuses the null context
    assert reached == [mako_attn.EINVAL]
    for key, t in ok.items():
        if not torch.is_tensor(t):
            continue
        for other in (torch.float32, torch.float64, torch.float16, torch.bfloat16, torch.int32, torch.int64, torch.uint8):
            first = "k" if name == "cache_evict" else "q"
            if other == t.dtype or (key == first and t.to(other).dtype in (torch.float16, torch.bfloat16)):
                continue
            with pytest.raises(TypeError):
                getattr(c, name)(**{**ok, key: t.to(other)})
    # one 16-bit type beside another
    with pytest.raises(TypeError):
        getattr(c, name)(**{**ok, "v": ok["v"].to(torch.bfloat16)})
    assert reached == [mako_attn.EINVAL]


def test_output_type_follows_the_option(monkeypatch):
    import mako_attn
    import torch
    c, calls = make()
    reached = []
    mako_attn._load_types()
    monkeypatch.setattr(mako_attn, "_raw_stream", lambda device: 0)
    monkeypatch.setattr(mako_attn, "_check", reached.append)
    for name in ("attention_tree", "attention_decode_weights"):
        ok = calls[name]
        for value, good, bad in ((1, torch.float16, torch.float32), (0, torch.float32, torch.float16)):
            c.set_option(mako_attn.OPT_OUTPUT_16BIT, value)
            getattr(c, name)(**{**ok, "o": ok["o"].to(good)})
            with pytest.raises(TypeError):
                getattr(c, name)(**{**ok, "o": ok["o"].to(bad)})


def test_too_few_frequencies():
    c, calls = make()
    ok = calls["cache_append"]
    with pytest.raises(ValueError, match="63 frequencies for 128"):
        c.cache_append(**{**ok, "freq": ok["freq"][:63]})


def test_masks_may_be_unsigned(monkeypatch):
    import mako_attn
    import torch
    c, calls = make()
    mako_attn._load_types()
    monkeypatch.setattr(mako_attn, "_raw_stream", lambda device: 0)
    reached = []
    monkeypatch.setattr(mako_attn, "_check", reached.append)
    c.attention_tree(**{**calls["attention_tree"], "mask": torch.zeros(4, dtype=torch.int32).view(torch.uint32)})
    assert reached == [mako_attn.EINVAL]
