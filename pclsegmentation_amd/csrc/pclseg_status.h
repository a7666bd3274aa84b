// pclseg_status.h — how the translation units beside pclseg_api.hip report a failure: the text goes where
// pclseg_last_error(NULL) reads it, the code is returned by the C entry point.
#ifndef PCLSEG_STATUS_H_
#define PCLSEG_STATUS_H_

#include <string>

namespace pclseg {

// records msg as the calling thread's last handle-less error and returns code (a pclseg_status)
int op_fail(int code, const std::string& msg);
// called inside a catch block of an extern "C" entry point: the exception in flight as a status (never throws)
int op_exception() noexcept;

}  // namespace pclseg

#endif  // PCLSEG_STATUS_H_
