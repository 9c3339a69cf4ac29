"""CPU check of the kernels' waits: what other blocks of a cluster stored with
st.async is read after a wait that acquires at the cluster's scope (a wait
without a scope acquires at the block's own, which orders nothing of theirs)."""
import os
import re

import autoresearch2_b200

CSRC = os.path.join(os.path.dirname(autoresearch2_b200.__file__), "csrc")


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def test_waits_for_stores_of_other_blocks_acquire_at_cluster_scope():
    users = [f for f in sorted(os.listdir(CSRC)) if f.endswith(".cu") and "st.async" in source(f)]
    assert users
    for name in users:
        waits = re.findall(r"mbar_(?:try_wait(?:_hint)?|wait_bounded)(<[^>]*>)?\(", source(name))
        assert waits and all(w == "<true>" for w in waits), name


def test_the_cluster_form_names_semantics_and_scope():
    forms = re.findall(r"mbarrier\.try_wait\.parity\S*", source("sm100.cuh"))
    assert len(forms) == 4 and sum("acquire.cluster" in f for f in forms) == 2
