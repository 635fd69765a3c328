"""What the 8-bit draft cache and the 4-bit head decide on the host, at the edges: workspaces sized once for many calls."""

import pytest

import kv8_cache
import mfd_hip


@pytest.mark.parametrize("bs,heads,group,modes,block", [(1, 8, 4, 1, 1), (1, 8, 4, 8, 16), (1, 8, 1, 8, 16), (4, 8, 4, 1, 1),
                                                        (4, 2, 4, 1, 16), (16, 8, 5, 1, 1), (65, 1, 3, 1, 1), (2, 8, 1, 8, 16)])
@pytest.mark.parametrize("splits", [-1, 0, 2, 3, 32, 64])
def test_a_workspace_serves_every_shorter_context(monkeypatch, bs, heads, group, modes, block, splits):
    """workspace_bytes for a longest context is enough for every call whose max_ctx is smaller, as one that the page table's reach
    cuts: the number of splits itself rises and falls with max_ctx."""
    monkeypatch.setattr(mfd_hip, "cu_count", lambda device: 256)
    sizes = dict(bs=bs, num_modes=modes, block_size=block, num_heads=heads * group, num_kv_heads=heads, with_block=True)
    lens = sorted({1, 63, 64, 65, 100001} | {x + d for x in range(128, 33000, 320) for d in (-1, 0, 1)}
                  | {2880, 2881, 16128, 16129, 2048, 2049})
    largest = 0
    for n in lens:
        if splits < 0:
            count, _ = kv8_cache._auto_splits(bs, heads, group * modes * block, True, n, None)
        else:
            count = kv8_cache._splits_of(splits, n)[0] if splits > 1 else 1
        need = mfd_hip.lib().mfd_kv8_attn_workspace_bytes(bs, modes, block, heads * group, heads, 1, count)
        largest = max(largest, need)
        assert kv8_cache.workspace_bytes(max_ctx=n, num_ctx_splits=splits, device="cuda:0", **sizes) >= largest, n


def test_a_workspace_for_no_requests(monkeypatch):
    monkeypatch.setattr(mfd_hip, "cu_count", lambda device: 256)
    for modes, block in ((1, 1), (8, 16)):
        for splits in (-1, 0, 4):
            assert kv8_cache.workspace_bytes(bs=0, num_modes=modes, block_size=block, num_heads=32, num_kv_heads=8,
                                             with_block=True, max_ctx=4096, num_ctx_splits=splits, device="cuda:0") == 0


def test_a_hidden_size_beyond_32_bit_offsets_is_refused():
    """The wide form addresses a workgroup's share of the weight, up to 672 rows of hidden / 2 bytes, by 32-bit offsets."""
    P, U8 = 1 << 20, 1 << 23  # (no pointer gets as far as being used)
    call = lambda K: mfd_hip.lib().mfd_draft_head_mxfp4(P, K, 1, K, P, P, 1, 100000, K, P, 100000, None)  # noqa: E731
    assert 672 * U8 // 2 < 2 ** 32 < 672 * 2 * U8 // 2
    for K in (U8 + 128, 2 * U8, 2 ** 31 - 128):
        assert call(K) == -2 and b"hidden" in mfd_hip.lib().mfd_last_error()
