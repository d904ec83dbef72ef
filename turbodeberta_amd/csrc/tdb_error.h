// The error text of the C ABI.
#pragma once

// Leaves the message that tdb_last_error() returns to this thread; returns the code.
int tdb_fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
