# Reads the compiler's resource remarks and fails where a kernel spills scalar
# registers, or where there are no remarks to read. A build of the attention
# that spilled them gave wrong results for 256 dimensions with a window; why was
# not found, so no such kernel is shipped.
/remark:.*Function Name:/ {
  name = $0
  sub(/.*Function Name: */, "", name)
  sub(/ *\[.*/, "", name)
}
/remark:.*SGPRs Spill:/ {
  ++seen
  count = $0
  sub(/.*SGPRs Spill: */, "", count)
  if (count + 0 > 0) {
    print name " spills " count + 0 " scalar registers"
    bad = 1
  }
}
END {
  if (!seen) print "no resource remarks"
  exit bad || !seen
}
