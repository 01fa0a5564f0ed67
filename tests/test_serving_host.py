"""What the operators around a serving step refuse, and their workspace sizes (no GPU: every refusal comes before anything is enqueued)."""
import ctypes as C

import numpy as np
import pytest

import nvr_import

nvr = nvr_import.load()
INVALID, UNSUPPORTED = -7, -8
P = 0x100000          # a pointer that is never followed: 1 MiB, aligned


def _status():
    import re
    text = open(nvr.HEADER_PATH).read()
    return {n: int(v) for n, v in re.findall(r"(NVR_ERR_\w+) = (-\d+)", text)}


STATUS = _status()


def refused(call, name, *args):
    rc = getattr(nvr.lib(), call)(*args)
    assert rc == STATUS[name], (rc, nvr.last_error())
    assert call in nvr.last_error()


@pytest.fixture(autouse=True)
def _type():
    nvr.check(nvr.lib().nvr_ops_set_dtype(b"float16"))
    yield


ROPE = dict(q=P, ldq=256, k=P, ldk=128, v=P, ldv=128, positions=P, slots=P, T=3, H=4, KVH=2, D=64, rotary=64, pairs=0, turns=P, amplitude=1.0, q_out=2 * P, ldqo=256, k_out=2 * P,
            ldko=128, k_cache=P, v_cache=P, num_slots=16, stream=None)


@pytest.mark.parametrize("change", [dict(T=-1), dict(H=-1), dict(H=0, KVH=0), dict(D=0), dict(rotary=0), dict(rotary=63), dict(rotary=66), dict(positions=None), dict(turns=None), dict(q=None),
                                    dict(q_out=None), dict(k=None), dict(k_cache=None), dict(v_cache=None), dict(slots=None), dict(v=None), dict(num_slots=-1), dict(ldq=255), dict(ldk=127),
                                    dict(ldv=127), dict(ldqo=255), dict(ldko=127), dict(k_out=None, k_cache=None, v_cache=None), dict(q_out=P, ldqo=512), dict(k_out=P, ldko=256),
                                    dict(D=2048, rotary=64), dict(H=1 << 40)])
def test_rope_refusals(change):
    refused("nvr_rope_rotate_store_kv", "NVR_ERR_INVALID_ARG", *{**ROPE, **change}.values())


def test_rope_of_more_tokens_than_a_launch_holds():
    refused("nvr_rope_rotate_store_kv", "NVR_ERR_UNSUPPORTED", *{**ROPE, "T": (1 << 23) + 1}.values())


def test_rope_of_no_rows_is_nothing():
    assert nvr.lib().nvr_rope_rotate_store_kv(*{**ROPE, "T": 0}.values()) == 0


@pytest.mark.parametrize("change", [dict(kind=5), dict(kind=-1), dict(theta=0.0), dict(theta=float("nan")), dict(kind=1, factor=0.0), dict(kind=1, factor=float("inf")), dict(kind=3, original_len=0.0),
                                    dict(kind=3, low=2.0, high=2.0), dict(kind=4, low=0.0), dict(kind=4, high=float("inf")), dict(kind=3, theta=1.0)])
def test_rope_frequencies_refusals(change):
    sc = nvr.RopeScalingC(**{**dict(kind=0, theta=1e4, factor=2.0, original_len=2048.0, low=1.0, high=4.0), **change})
    refused("nvr_rope_frequencies", "NVR_ERR_INVALID_ARG", C.byref(sc), 64, P, C.byref(C.c_float()))


@pytest.mark.parametrize("rotary", [0, -2, 63, 4098])
def test_rope_frequencies_refuse_odd_parts(rotary):
    sc = nvr.RopeScalingC(0, 1e4, 1.0, 0, 0, 0)
    refused("nvr_rope_frequencies", "NVR_ERR_INVALID_ARG", C.byref(sc), rotary, P, C.byref(C.c_float()))
    refused("nvr_rope_frequencies", "NVR_ERR_INVALID_ARG", None, 64, P, C.byref(C.c_float()))
    refused("nvr_rope_frequencies", "NVR_ERR_INVALID_ARG", C.byref(sc), 64, None, C.byref(C.c_float()))


LORA = dict(x=P, ldx=64, A=P, B=P, scales=P, ids=P, n=3, T=5, K=64, N=32, R=8, base=P, ldb=32, y=2 * P, ldy=32, ws=P, stream=None)


@pytest.mark.parametrize("change,name", [(dict(T=-1), "NVR_ERR_INVALID_ARG"), (dict(K=0), "NVR_ERR_INVALID_ARG"), (dict(N=0), "NVR_ERR_INVALID_ARG"), (dict(R=0), "NVR_ERR_INVALID_ARG"),
                                         (dict(n=-1), "NVR_ERR_INVALID_ARG"), (dict(R=257), "NVR_ERR_UNSUPPORTED"), (dict(n=8192), "NVR_ERR_UNSUPPORTED"), (dict(x=None), "NVR_ERR_INVALID_ARG"),
                                         (dict(A=None), "NVR_ERR_INVALID_ARG"), (dict(B=None), "NVR_ERR_INVALID_ARG"), (dict(ids=None), "NVR_ERR_INVALID_ARG"),
                                         (dict(base=None), "NVR_ERR_INVALID_ARG"), (dict(y=None), "NVR_ERR_INVALID_ARG"), (dict(ws=None), "NVR_ERR_INVALID_ARG"),
                                         (dict(ws=P + 8), "NVR_ERR_INVALID_ARG"), (dict(ldx=63), "NVR_ERR_INVALID_ARG"), (dict(ldb=31), "NVR_ERR_INVALID_ARG"),
                                         (dict(ldy=31), "NVR_ERR_INVALID_ARG"), (dict(y=P, ldy=40), "NVR_ERR_INVALID_ARG"), (dict(K=1 << 40, ldx=1 << 40), "NVR_ERR_UNSUPPORTED")])
def test_lora_refusals(change, name):
    refused("nvr_lora_add", name, *{**LORA, **change}.values())


@pytest.mark.parametrize("change", [dict(T=(1 << 19) + 1), dict(N=(1 << 22) + 1, ldb=1 << 23, ldy=1 << 23), dict(K=(1 << 22) + 1, ldx=1 << 23)])
def test_lora_sizes_that_no_grid_holds(change):
    refused("nvr_lora_add", "NVR_ERR_UNSUPPORTED", *{**LORA, **change}.values())


def test_lora_of_no_rows_or_adapters_is_nothing():
    assert nvr.lib().nvr_lora_add(*{**LORA, "T": 0}.values()) == 0
    assert nvr.lib().nvr_lora_add(*{**LORA, "n": 0, "A": None, "B": None, "y": P}.values()) == 0     # in place, no adapter: every row stays


SAMPLE = dict(logits=P, ld=100, B=4, V=100, T=P, k=P, p=P, m=P, u=P, ids=P, logprobs=P, ws=P, stream=None)


@pytest.mark.parametrize("change,name", [(dict(B=-1), "NVR_ERR_INVALID_ARG"), (dict(V=0), "NVR_ERR_INVALID_ARG"), (dict(ld=99), "NVR_ERR_INVALID_ARG"), (dict(logits=None), "NVR_ERR_INVALID_ARG"),
                                         (dict(u=None), "NVR_ERR_INVALID_ARG"), (dict(ids=None), "NVR_ERR_INVALID_ARG"), (dict(ws=None), "NVR_ERR_INVALID_ARG"), (dict(ws=P + 4), "NVR_ERR_INVALID_ARG"),
                                         (dict(V=(1 << 22) + 1, ld=1 << 23), "NVR_ERR_UNSUPPORTED"), (dict(B=65536), "NVR_ERR_UNSUPPORTED")])
def test_sample_refusals(change, name):
    refused("nvr_sample_uniform", name, *{**SAMPLE, **change}.values())


def _meta(**kw):
    return nvr.AttnMetaC(**{**dict(is_prefill=0, context_lens=P, block_tables=P, max_blocks=4, batch=2, max_context_len=50), **kw})


SCORED = dict(q=P, ldq=256, k=P, v=P, meta=None, H=4, KVH=2, D=64, bs=16, nb=8, scale=0.125, scores=P, scored=P, decay=1.0, new=P, out=P, ws=P, stream=None)


@pytest.mark.parametrize("change,name", [(dict(H=3), "NVR_ERR_INVALID_ARG"), (dict(H=0), "NVR_ERR_INVALID_ARG"), (dict(KVH=0), "NVR_ERR_INVALID_ARG"), (dict(bs=0), "NVR_ERR_INVALID_ARG"),
                                         (dict(nb=-1), "NVR_ERR_INVALID_ARG"), (dict(D=96, ldq=384), "NVR_ERR_UNSUPPORTED"), (dict(H=34, ldq=34 * 64), "NVR_ERR_UNSUPPORTED"),
                                         (dict(nb=1 << 30), "NVR_ERR_UNSUPPORTED"), (dict(nb=1 << 40), "NVR_ERR_INVALID_ARG"), (dict(q=None), "NVR_ERR_INVALID_ARG"),
                                         (dict(k=None), "NVR_ERR_INVALID_ARG"), (dict(v=P + 2), "NVR_ERR_INVALID_ARG"), (dict(scores=None), "NVR_ERR_INVALID_ARG"),
                                         (dict(new=None), "NVR_ERR_INVALID_ARG"), (dict(out=None), "NVR_ERR_INVALID_ARG"), (dict(ws=None), "NVR_ERR_INVALID_ARG"), (dict(ldq=255), "NVR_ERR_INVALID_ARG")])
def test_scored_attention_refusals(change, name):
    m = _meta()
    refused("nvr_paged_attn_decode_scored", name, *{**SCORED, "meta": C.byref(m), **change}.values())


def test_scored_attention_refuses_missing_metadata():
    refused("nvr_paged_attn_decode_scored", "NVR_ERR_INVALID_ARG", *SCORED.values())
    for kw in (dict(context_lens=None), dict(block_tables=None), dict(batch=-1), dict(max_context_len=-1), dict(max_blocks=-1)):
        refused("nvr_paged_attn_decode_scored", "NVR_ERR_INVALID_ARG", *{**SCORED, "meta": C.byref(_meta(**kw))}.values())
    assert nvr.lib().nvr_paged_attn_decode_scored(*{**SCORED, "meta": C.byref(_meta(batch=0))}.values()) == 0


EVICT = dict(k=P, v=P, scores=P, meta=None, KVH=2, D=64, bs=16, nb=8, budget=32, first=4, last=8, to=None, to_blocks=0, new_lens=2 * P, kept=P, ws=P, stream=None)


@pytest.mark.parametrize("change,name", [(dict(KVH=0), "NVR_ERR_INVALID_ARG"), (dict(D=0), "NVR_ERR_INVALID_ARG"), (dict(bs=0), "NVR_ERR_INVALID_ARG"), (dict(budget=0), "NVR_ERR_INVALID_ARG"),
                                         (dict(first=-1), "NVR_ERR_INVALID_ARG"), (dict(last=-1), "NVR_ERR_INVALID_ARG"), (dict(first=20, last=13), "NVR_ERR_INVALID_ARG"),
                                         (dict(D=4), "NVR_ERR_UNSUPPORTED"), (dict(D=1024), "NVR_ERR_UNSUPPORTED"), (dict(nb=1 << 30), "NVR_ERR_UNSUPPORTED"), (dict(k=None), "NVR_ERR_INVALID_ARG"),
                                         (dict(k=P + 8), "NVR_ERR_INVALID_ARG"), (dict(scores=None), "NVR_ERR_INVALID_ARG"), (dict(new_lens=None), "NVR_ERR_INVALID_ARG"),
                                         (dict(new_lens=P), "NVR_ERR_INVALID_ARG"), (dict(to=P), "NVR_ERR_INVALID_ARG"), (dict(kept=None, ws=None), "NVR_ERR_INVALID_ARG")])
def test_evict_refusals(change, name):
    m = _meta()
    refused("nvr_kv_evict", name, *{**EVICT, "meta": C.byref(m), **change}.values())


def test_evict_refuses_missing_metadata():
    refused("nvr_kv_evict", "NVR_ERR_INVALID_ARG", *EVICT.values())
    refused("nvr_kv_evict", "NVR_ERR_INVALID_ARG", *{**EVICT, "meta": C.byref(_meta(block_tables=None))}.values())
    assert nvr.lib().nvr_kv_evict(*{**EVICT, "meta": C.byref(_meta(batch=0))}.values()) == 0


def test_workspace_sizes_grow_with_the_work():
    l = nvr.lib()
    assert l.nvr_lora_workspace_bytes(0, 64, 64, 8) == 0 and l.nvr_sample_uniform_workspace_bytes(0, 10) == 0 and l.nvr_kv_evict_workspace_bytes(1, 1, 0, 10) == 0
    assert l.nvr_paged_attn_scored_workspace_bytes(1, 4, 2, 64, 0) == 0
    for T in (1, 255, 256, 257, 5000):
        assert l.nvr_lora_workspace_bytes(T, 4096, 64, 20) >= T * 32 * 4
    assert l.nvr_kv_evict_workspace_bytes(3, 2, 100, 1000) >= 3 * 2 * 100 * 4
    for B, n in ((1, 1), (1, 100000), (64, 5000)):
        assert l.nvr_paged_attn_scored_workspace_bytes(B, 8, 2, 128, n) >= B * 8 * (n + 130) * 4


def test_definitions_agree_with_hand_computed_cases():
    """The 64-bit definitions of serving_util themselves."""
    import serving_util as su
    assert su.sample(np.log([0.5, 0.3, 0.2]), 1.0, 0, 1.0, 0.0, 0.6)[0] == 1
    assert su.sample(np.log([0.2, 0.3, 0.5]), 1.0, 2, 1.0, 0.0, 0.3)[0] == 1                # 0.375 and 0.625 in index order
    assert su.sample(np.zeros(4), 1.0, 0, 0.5, 0.0, 0.9)[0] == 1                            # the first two of four equal ones
    assert su.sample(np.log([0.5, 0.26, 0.24]), 1.0, 0, 1.0, 0.5, 0.99)[0] == 1
    assert su.evict(np.array([9.0, 1.0, 3.0, 3.0, 0.0, 5.0]), 4, 1, 1).tolist() == [0, 2, 3, 5]
    x = np.arange(8.0).reshape(1, 1, 8)
    turns = np.array([0.25, 0.0])
    assert np.allclose(su.rope(x, np.array([1]), turns, 1.0, False)[0, 0], [-2, 1, 0, 3, 4, 5, 6, 7])
    assert np.allclose(su.rope(x, np.array([1]), turns, 1.0, True)[0, 0], [-1, 0, 2, 3, 4, 5, 6, 7])


def test_workspaces_of_larger_steps_serve_smaller_ones():
    """A program allocates once, for its largest step: no size falls where rows, columns, keys or a budget grow, also where a rule on sizes changes what the kernels do."""
    l = nvr.lib()
    rows = [1, 2, 63, 64, 65, 126, 127, 128, 129, 255, 256, 257, 512, 1000, 1024, 1025, 4000, 65535]
    logits = [1, 33, 4095, 4096, 4097, 5000, 10000, 16383, 16384, 16385, 20570, 65536, 98303, 98304, 98305, 114688, 114689, 151936, 400000, (1 << 22) - 1, 1 << 22]
    keys = [1, 127, 128, 129, 255, 256, 257, 511, 512, 513, 4096, 8100, 65536, 1 << 20, 1 << 23]
    wide = [8, 511, 512, 1023, 1024, 1535, 1536, 2047, 2048, 4096, 1 << 16, 1 << 22]
    grids = {"nvr_sample_uniform_workspace_bytes": [(rows, logits)],
             "nvr_lora_workspace_bytes": [(rows + [1 << 17, 1 << 19], wide, [n], [1, 15, 16, 17, 64, 96, 97, 128, 129, 256]) for n in (8, 4096)],
             "nvr_paged_attn_scored_workspace_bytes": [(rows, [h], [g], [d], keys) for h, g in ((1, 1), (32, 8), (16, 1), (64, 64)) for d in (64, 128, 256)],
             "nvr_kv_evict_workspace_bytes": [(rows, [1, 8], [1, 16, 2048, 1 << 20], keys)]}
    for name, all_axes in grids.items():
        for axes in all_axes:
            size = np.zeros([len(a) for a in axes], np.float64)
            for at in np.ndindex(*size.shape):
                size[at] = getattr(l, name)(*(int(a[i]) for a, i in zip(axes, at)))
            assert (size > 0).all()
            for d in range(size.ndim):
                fell = np.argwhere(np.diff(size, axis=d) < 0)
                assert len(fell) == 0, (name, "argument", d, [a[i] for a, i in zip(axes, fell[0])])


@pytest.mark.parametrize("kw,bs,name", [(dict(max_context_len=(1 << 25) + 1, max_blocks=1 << 22), 16, "NVR_ERR_UNSUPPORTED"), (dict(max_context_len=2 ** 31 - 1, max_blocks=2 ** 31 - 1), 1, "NVR_ERR_UNSUPPORTED"),
                                        (dict(max_context_len=2 ** 31 - 1, max_blocks=(1 << 23) + 1), 256, "NVR_ERR_UNSUPPORTED"), (dict(max_context_len=2 ** 31 - 1, max_blocks=3), 1 << 24, "NVR_ERR_UNSUPPORTED")])
def test_evict_refuses_contexts_that_no_launch_holds(kw, bs, name):
    """Tables and bound together allow more than 2^25 keys: sums of 32 bits over a sequence's blocks, and the grid of the copy, would pass their ends."""
    refused("nvr_kv_evict", name, *{**EVICT, "nb": 8, "bs": bs, "meta": C.byref(_meta(**kw))}.values())
