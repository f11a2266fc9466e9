"""CPU checks of the largest calls of paged attention: what would pass 2^32 threads in a launch is
refused, and one tile or sequence less is not (the call then ends at its missing workspace)."""
import pytest

from localmoe35ba3b_amd import _lib
from tests.test_cache8_checks import c_call


def attend(eight, **change):
    """A call without a workspace, of a cache of 8 or 16 bits."""
    size = dict(ws=None, page_stride=change['k_heads'] * 16 * change['dim'],
                scale_stride=2 * change['k_heads'], q_token=change['q_heads'] * change['dim'],
                q_head=change['dim'], **change)
    if eight:
        return c_call('attend8', **size)
    at = 4096
    rc = _lib.lib().lm_paged_attention(
        at, size['q_token'], size['q_head'], size['q_heads'], at, at, 6, size['page_stride'],
        size['k_heads'], 16, size['dim'], at, at, at, 3, size.get('table_pages', 3), size['sequences'],
        size['tokens'], size['max_new'], 0.1, None, 0, 0, at, None, 0, 0, None)
    return rc, _lib.lib().lm_last_error().decode()


@pytest.mark.parametrize('eight,tokens,message', [
    (True, 131024, 'too many rows'), (True, 131008, 'workspace'), (False, 131024, 'workspace'),
    (False, 131040, 'too many rows')])
def test_tiles_and_few_rows_in_one_launch(eight, tokens, message):
    """Heads of 256: 512 threads a workgroup; over 8 bits the few rows' workgroups go along."""
    rc, error = attend(eight, tokens=tokens, max_new=tokens, sequences=2, q_heads=8192, k_heads=1024,
                       dim=256)
    assert rc == _lib.LM_EINVAL and message in error


@pytest.mark.parametrize('eight', [False, True])
@pytest.mark.parametrize('sequences,message', [(61455, 'too many rows'), (61450, 'workspace')])
def test_joining_parts_of_both_kinds(eight, sequences, message):
    """A workgroup for each sequence's key-value head, and those of the tokens whose tiles are split."""
    rc, error = attend(eight, tokens=3, max_new=3, sequences=sequences, q_heads=1638, k_heads=273,
                       dim=128, table_pages=64)
    assert rc == _lib.LM_EINVAL and message in error
