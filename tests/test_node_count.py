"""A node count past 64 bits is no number: refused, where it used to fill the memory with hostnames."""

import io

import pytest
import yaml

from test_cli_fuzz import CLUSTER, DOCS, NODE

from triton_kubernetes_amd.cli.main import run


@pytest.mark.parametrize("count", ["99999999999999999999", 1 << 63])
@pytest.mark.parametrize("cmd", ["cluster", "node"])
def test_a_count_past_64_bits_is_refused(tk_home, tmp_path, cmd, count):
    manager = tk_home / ".triton-kubernetes" / "m"
    manager.mkdir(parents=True)
    (manager / "main.tf.json").write_text('{"module": {"cluster-manager": {"name": "m"}, '
                                          '"cluster_baremetal_c": {"name": "c"}}}')
    doc = dict(DOCS[("create", "node")], node_count=count) if cmd == "node" else \
        dict(CLUSTER, name="d", nodes=[dict(NODE, node_count=count)])
    path = tmp_path / "c.yaml"
    path.write_text(yaml.safe_dump(doc))
    out = io.StringIO()
    assert run(["--non-interactive", "--config", str(path), "create", cmd], out=out) == 1
    assert "node_count must be a valid number" in out.getvalue()
