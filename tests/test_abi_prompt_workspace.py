"""Each form of the prompt attention asks for the workspace that it uses, without a GPU."""
from test_abi_paged import lib  # noqa: F401


def test_each_form_asks_for_its_own(lib):  # noqa: F811
    plain, eight = lib.moss_paged_prompt_workspace_bytes, lib.moss_paged_prompt_workspace_bytes_fp8
    # 2500 tokens of 4 heads a KV head, up to 16000 rows: 64 parts of the 32 shares' for 8 KV heads, tiles of 64 and 128 rows
    assert plain(1, 1000, 16, 2500, 32, 8, 128) == 64 * 8 * 64 * 130 * 4
    assert eight(1, 1000, 16, 2500, 32, 8, 128) == 64 * 8 * 128 * 130 * 4
    # few tiles and many: the same tiles in both
    for tokens in (1, 45, 512, 2048, 4097, 8000):
        assert plain(1, 1000, 16, tokens, 32, 8, 128) == eight(1, 1000, 16, tokens, 32, 8, 128) > 0
    for shape in ((1, 4, 16, 2500, 32, 8, 128), (0, 4, 16, 50, 32, 8, 128), (3, 100, 16, 0, 32, 8, 128), (3, 100, 16, 50, 32, 8, 80)):
        assert plain(*shape) == eight(*shape) == 0


def test_no_shape_asks_for_less_in_8_bits(lib):  # noqa: F811
    for b in (1, 3, 40, 700):
        for w in (1, 33, 40, 5000):
            for tokens in (1, 31, 300, 700, 1100, 2500, 4097, 20000):
                for heads in ((32, 8, 128), (12, 12, 64), (16, 1, 128), (28, 4, 128)):
                    shape = b, w, 16, tokens, *heads
                    assert lib.moss_paged_prompt_workspace_bytes(*shape) <= lib.moss_paged_prompt_workspace_bytes_fp8(*shape) <= \
                        2 * lib.moss_paged_prompt_workspace_bytes(*shape)
