"""Workspaces of the operators on drafted trees (no device): what is asked for, and what a
given length is used for."""
import pytest

from compiler_amd import runtime as rt
from test_abi_tree import attend, verify


def verify_parts(b, v):
    """Workgroups of a sequence where the workspace has places for them (256 CUs)."""
    return max(1, min(512 // b, v // 2048, 64))


@pytest.mark.parametrize("b,t,v", [(1, 26, 32000), (1, 61, 128000), (1, 1024, 32000), (16, 16 * 26, 128000),
                                   (4, 4 * 200, 50257), (2, 33, 4096), (300, 9000, 128000), (3, 0, 4096)])
def test_verification_has_places_for_every_sum(b, t, v):
    """A refusal takes a sum, so a tree of n nodes can need n of them from each workgroup."""
    got, parts = rt.load_library().g950_verify_tree_workspace(None, b, t, v), verify_parts(b, v)
    assert got == 0 if parts == 1 else got >= 16 * t + 8 * parts * t


def test_a_workspace_short_of_places_means_fewer_workgroups():
    """Two workgroups for a tree of 200 nodes: 16 bytes a node, and a place a node for each."""
    need = (16 * 200 + 8 * 2 * 200) // 4
    assert verify(t=200, b=1, vocab=6000, ws=need)[1] == "g950_verify_tree_f32_parts"
    assert verify(t=200, b=1, vocab=6000, ws=need - 1)[1] == "g950_verify_tree_f32"


@pytest.mark.parametrize("b,h,hk,d,nodes,keys,parts,blocks,rows", [
    (32, 32, 8, 128, 1, 4096, 192, 8, 4),       # a decoding step: four rows a KV head
    (1, 32, 8, 128, 26, 1000, 64, 8, 104),
    (8, 32, 8, 128, 64, 8192, 32, 16, 128),     # two blocks of 128 rows a KV head
    (2, 8, 1, 64, 13, 65537, 256, 1, 104), (1, 8, 8, 256, 1, 1000, 128, 8, 1), (3, 8, 2, 64, 1, 512, 0, 2, 4)])
def test_attention_records_hold_the_rows_that_there_are(b, h, hk, d, nodes, keys, parts, blocks, rows):
    """O, maximum and sum in fp32 of each part's rows, none of the rows that no tree of the batch has."""
    got = rt.load_library().g950_paged_attention_tree_workspace(None, b, h, hk, d, nodes, keys)
    assert got == parts * blocks * rows * (d + 2) * 4


def test_a_workspace_of_two_records_makes_two_parts():
    kw = dict(b=1, t=1, h=8, hk=2, sq=1, sk=4000)
    assert attend(ws=2 * 2 * 4 * 130, **kw)[1] == "g950_attn_tree_bf16_d128_r2_merge16"
    assert attend(ws=2 * 2 * 4 * 130 - 1, **kw)[1] == "g950_attn_tree_bf16_d128_r2"
